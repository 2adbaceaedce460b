"""Workloads of the attention operators: per-head norm with rotation, cross attention, the 8-bit state cache.

``listed()`` names the measured cases, ``draw(rng)`` gives further ones of the
same ranges, ``prepare`` makes what a caller has in hand, ``run`` is one pass.
With ``own`` false the pass is the plain form (elementary torch operations in
fp32, rounded once at the end); with ``own`` true it is the call a user makes
of hclsm_b200.  ``exact`` is the definition in 64 bits.
"""
import math

import torch

own = False

F32 = torch.float32


# ---- the cases ----------------------------------------------------------------------------------
def _rope(name, B, Lq, Lk, H, Hkv, D, R, *, dtype="bf16", train=True, inter=False, weight=True):
    return {"name": name, "op": "rope", "B": B, "Lq": Lq, "Lk": Lk, "H": H, "Hkv": Hkv, "D": D, "R": R,
            "dtype": dtype, "train": train, "inter": inter, "weight": weight}


def _xattn(name, B, Lq, Lk, H, Hkv, D, *, dtype="bf16", train=True, ragged=False, mask=False):
    return {"name": name, "op": "xattn", "B": B, "Lq": Lq, "Lk": Lk, "H": H, "Hkv": Hkv, "D": D,
            "dtype": dtype, "train": train, "ragged": ragged, "mask": mask}


def _kv8(name, op, B, T, n, H, Hkv, D, *, block=32, dtype="bf16"):
    return {"name": name, "op": op, "B": B, "T": T, "n": n, "H": H, "Hkv": Hkv, "D": D, "block": block,
            "dtype": dtype}


def listed():
    return [
        # one rollout step: a single goal query and a single new state per video, 6 heads of 64
        _rope("rope_step", 8, 1, 1, 6, 6, 64, 64, train=False),
        # Level-1 widths (d 384): 32 slots attending to the 64 x 32 states of 8 videos, fp32 module
        _rope("rope_events_f32", 8, 32, 2048, 6, 6, 64, 32, dtype="f32", inter=True),
        # base width (d 2048 as 32 heads of 64, 8 shared key heads), 64 videos, a training step
        _rope("rope_base_train", 64, 2048, 2048, 32, 8, 64, 64),
        # 32 slots of a frame attend to its 196 patch tokens, 8 x 16 frames, d 384 (training)
        _xattn("slots_tokens_train", 128, 32, 196, 6, 6, 64),
        # slots attend to the gathered events of their video: ragged event counts, dead slots (training)
        _xattn("goals_events_train", 8, 128, 2048, 6, 6, 64, ragged=True, mask=True),
        # the same call from an fp32 module, odd sizes
        _xattn("odd_train_f32", 3, 333, 777, 6, 2, 64, dtype="f32", ragged=True),
        # a long history at base width, shared key heads (training)
        _xattn("history_train", 8, 2048, 4096, 16, 4, 128),
        # histories of unequal lengths read without gradients, heads of 64, no sharing
        _xattn("history_eval", 4, 2048, 8192, 32, 32, 64, train=False, ragged=True),
        # one query token over a long history
        _xattn("history_step", 8, 1, 16384, 16, 4, 128, train=False, ragged=True),
        # the encoder's states of 8 videos written into the cache and read back
        _kv8("cache_fill", "fill", 8, 2048, 2048, 6, 6, 64),
        # a rollout step: one state appended to the cache, one query over it
        _kv8("cache_step", "step", 8, 2048, 1, 6, 6, 64),
        # the same over a long history at base width, shared key heads
        _kv8("cache_step_long", "step", 16, 65536, 1, 32, 8, 128),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(c):
    """Bytes or operations that the plain form goes through, to keep drawn cases below the listed ones."""
    B, H, D = c["B"], c["H"], c["D"]
    if c["op"] == "rope":
        return B * (c["Lq"] * H + c["Lk"] * c["Hkv"]) * D / (64 * 2048 * 40 * 64)
    if c["op"] == "xattn":
        return B * H * c["Lq"] * c["Lk"] * D * (3.5 if c["train"] else 1) / (8 * 16 * 2048 * 4096 * 128 * 3.5)
    return B * c["T"] * c["Hkv"] * D / (16 * 65536 * 8 * 128)


def draw(rng):
    while True:
        dtype = "f32" if rng.random() < 0.25 else "bf16"
        B, Hkv, G = _log(rng, 1, 64), _log(rng, 1, 12), rng.choice([1, 1, 2, 4, 5, 8])
        op = rng.choice(["rope", "xattn", "xattn", "xattn", "fill", "step"])
        if op == "rope":
            D = rng.choice([32, 64, 96, 128])
            c = _rope("", B, _log(rng, 1, 4096), _log(rng, 1, 4096), Hkv * G, Hkv, D, rng.choice([D, D // 2]),
                      dtype=dtype, train=rng.random() < 0.6, inter=rng.random() < 0.5, weight=rng.random() < 0.8)
        elif op == "xattn":
            one = rng.random() < 0.25
            c = _xattn("", B, 1 if one else _log(rng, 2, 4096), _log(rng, 16, 16384 if one else 8192), Hkv * G, Hkv,
                       rng.choice([32, 64, 64, 96, 128]), dtype=dtype, train=not one and rng.random() < 0.6,
                       ragged=rng.random() < 0.5, mask=rng.random() < 0.25)
            if dtype == "f32" and _cost(c) > 0.1:
                continue
        else:
            block = rng.choice([16, 32, 64])
            T = max(1, _log(rng, 64, 65536 if op == "step" else 4096) // block) * block
            c = _kv8("", op, B, T, T if op == "fill" else rng.choice([1, 1, 1, 32]), Hkv * G, Hkv,
                     rng.choice([32, 64, 128]), block=block, dtype=dtype)
            if op == "fill":
                c["H"] = Hkv
            elif c["n"] > 1 and _cost(c) * G > 0.25:
                continue
        if _cost(c) <= 1 and _scores(c) <= 1 << 31:
            del c["name"]
            return c


def _scores(c):
    """Scores that the plain form holds at once."""
    if c["op"] == "xattn":
        return c["B"] * c["H"] * c["Lq"] * c["Lk"]
    return c["B"] * c["H"] * c["n"] * c["T"] if c["op"] == "step" else 0


# ---- inputs ---------------------------------------------------------------------------------------
def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else F32


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _dtype(case)
    B, H, Hkv, D = case["B"], case["H"], case["Hkv"], case["D"]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=F32).to(dt)

    def ints(lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=g, device="cuda", dtype=torch.int32)

    s = {"case": case}
    if case["op"] == "rope":
        Lq, Lk, R = case["Lq"], case["Lk"], case["R"]
        P = max(Lq, Lk) + 64
        freq = 10000.0 ** (-torch.arange(0, R, 2, device="cuda", dtype=torch.float64) / R)
        ang = torch.arange(P, device="cuda", dtype=torch.float64)[:, None] * freq
        s["cos"], s["sin"] = ang.cos().float(), ang.sin().float()
        # queries and keys sit at different times of their videos
        s["q_pos"] = (ints(0, 64, B, 1) + torch.arange(Lq, device="cuda", dtype=torch.int32)).contiguous()
        s["k_pos"] = (ints(0, 64, B, 1) + torch.arange(Lk, device="cuda", dtype=torch.int32)).contiguous()
        s["q"], s["k"] = randn(B, Lq, H, D), randn(B, Lk, Hkv, D)
        for n in ("qw", "kw"):
            s[n] = 1.0 + 0.1 * torch.randn(D, generator=g, device="cuda") if case["weight"] else None
        if case["train"]:
            s["dq"], s["dk"] = randn(B, Lq, H, D), randn(B, Lk, Hkv, D)
        leaves = ("q", "k", "qw", "kw")
    elif case["op"] == "xattn":
        Lq, Lk = case["Lq"], case["Lk"]
        s["q"], s["k"], s["v"] = randn(B, Lq, H, D), randn(B, Lk, Hkv, D), randn(B, Lk, Hkv, D)
        s["lens"] = ints(Lk // 2, Lk + 1, B) if case["ragged"] else None
        # a tenth of the states are dead slots
        s["mask"] = torch.rand(B, Lk, generator=g, device="cuda") > 0.1 if case["mask"] else None
        if case["train"]:
            s["do"] = randn(B, Lq, H, D)
        leaves = ("q", "k", "v")
    else:
        T, n, block = case["T"], case["n"], case["block"]
        nb = T // block
        s["k"], s["v"] = randn(B, n, Hkv, D), randn(B, n, Hkv, D)
        for x in ("k", "v"):
            if case["op"] == "fill":
                s[x + "8"] = torch.zeros(B, Hkv, T, D, dtype=torch.int8, device="cuda")
                s[x + "s"] = torch.zeros(B, Hkv, nb, device="cuda")
            else:
                s[x + "8"] = torch.randint(-127, 128, (B, Hkv, T, D), generator=g, device="cuda", dtype=torch.int8)
                s[x + "s"] = (3.0 + torch.rand(B, Hkv, nb, generator=g, device="cuda")) / 127.0 / 2.0
            s[x + "t"] = randn(B, Hkv, block, D)
        if case["op"] == "fill":
            s["start"] = torch.zeros(B, dtype=torch.int32, device="cuda")
            s["count"] = ints(n // 2, n + 1, B)
        else:
            s["q"] = randn(B, n, H, D)
            s["start"] = ints(T // 2, T - n + 1, B)
            if n > 1:  # a whole step's states: sequences stand at a block's first token
                s["start"] = s["start"] // block * block
            s["count"] = torch.full((B,), n, dtype=torch.int32, device="cuda")
        s["total"] = s["start"] + s["count"]
        leaves = ()
    if case.get("train"):
        for n in leaves:
            if s[n] is not None:
                s[n].requires_grad_()
    return s


# ---- one pass ---------------------------------------------------------------------------------------
def run(s):
    op = s["case"]["op"]
    if op == "rope":
        return _rope_own(s) if own else _rope_plain(s)
    if op == "xattn":
        return _xattn_own(s) if own else _xattn_plain(s)
    return _kv8_own(s) if own else _kv8_plain(s)


def _rope_own(s):
    from hclsm_b200.kernels import qk_norm_rope

    q, k = qk_norm_rope(s["q"], s["k"], s["qw"], s["kw"], s["cos"], s["sin"], q_pos=s["q_pos"], k_pos=s["k_pos"],
                        interleaved=s["case"]["inter"])
    if not s["case"]["train"]:
        return {"q": q, "k": k}
    names = [n for n in ("q", "k", "qw", "kw") if s[n] is not None]
    grads = torch.autograd.grad((q, k), [s[n] for n in names], (s["dq"], s["dk"]))
    return {"q": q.detach(), "k": k.detach(), **{"d" + n: g for n, g in zip(names, grads)}}


def _xattn_own(s):
    from hclsm_b200.kernels import cross_attention

    o = cross_attention(s["q"], s["k"], s["v"], kv_lens=s["lens"], key_mask=s["mask"])
    if not s["case"]["train"]:
        return {"o": o}
    dq, dk, dv = torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["do"])
    return {"o": o.detach(), "dq": dq, "dk": dk, "dv": dv}


def _kv8_own(s):
    from hclsm_b200.kernels import Kv8Cache, kv8_attention, kv8_read, kv8_write

    cache = Kv8Cache(s["k8"], s["v8"], s["ks"], s["vs"], s["kt"], s["vt"])
    kv8_write(cache, s["k"], s["v"], s["start"], s["count"])
    if s["case"]["op"] == "fill":
        k, v = kv8_read(cache, s["total"])
        return {"k": k, "v": v, "kt": s["kt"], "vt": s["vt"]}
    return {"o": kv8_attention(s["q"], cache, s["total"]), "kt": s["kt"], "vt": s["vt"]}


def _rotate(x, cos, sin, inter):
    """The rotation of the first 2 * cos.shape[-1] dims by the given angles; x (B, L, H, D), cos (B, L, 1, R/2)."""
    R = 2 * cos.shape[-1]
    r, rest = x[..., :R], x[..., R:]
    if inter:
        a, b = r[..., 0::2], r[..., 1::2]
        y = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = r[..., :R // 2], r[..., R // 2:]
        y = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((y, rest), -1)


def _rope_one(x, w, cos, sin, pos, inter, dy):
    """(y, dx, dw) of one of the two tensors, dx and dw None without dy."""
    dt = x.dtype
    x = x.float()
    c, n = cos[pos.long()].unsqueeze(2), sin[pos.long()].unsqueeze(2)
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)
    xh = x * r
    y = _rotate(xh if w is None else xh * w, c, n, inter).to(dt)
    if dy is None:
        return y, None, None
    u = _rotate(dy.float(), c, -n, inter)
    dw = None if w is None else (u * xh).sum((0, 1, 2))
    gx = u if w is None else u * w
    dx = r * (gx - xh * (gx * xh).mean(-1, keepdim=True))
    return y, dx.to(dt), dw


@torch.no_grad()
def _rope_plain(s):
    inter = s["case"]["inter"]
    q, dq, dqw = _rope_one(s["q"], s["qw"], s["cos"], s["sin"], s["q_pos"], inter, s.get("dq"))
    k, dk, dkw = _rope_one(s["k"], s["kw"], s["cos"], s["sin"], s["k_pos"], inter, s.get("dk"))
    out = {"q": q, "k": k}
    if s["case"]["train"]:
        out.update(dq=dq, dk=dk)
        if dqw is not None:
            out.update(dqw=dqw, dkw=dkw)
    return out


def _heads(x, Hkv):
    """(B, L, H, D) as (B, Hkv, H / Hkv * L, D) in fp32: the query heads that share a key head, one after another."""
    B, L, H, D = x.shape
    return x.float().permute(0, 2, 1, 3).reshape(B, Hkv, H // Hkv * L, D)


def _tokens(x, L, H):
    """The inverse of _heads."""
    B, D = x.shape[0], x.shape[-1]
    return x.reshape(B, H, L, D).permute(0, 2, 1, 3)


def _softmax(scores, allowed):
    """Row softmax over the allowed keys (allowed: broadcast over scores or None); zero rows where none is."""
    if allowed is not None:
        scores = scores.masked_fill(~allowed, -torch.inf)
    m = scores.amax(-1, keepdim=True)
    if allowed is not None:
        m = torch.where(m > -torch.inf, m, 0.0)
    p = torch.exp(scores - m)
    z = p.sum(-1, keepdim=True)
    return p / (z if allowed is None else torch.where(z > 0, z, 1.0))


@torch.no_grad()
def _xattn_plain(s):
    c, dt = s["case"], s["q"].dtype
    H, Hkv, Lq, Lk = c["H"], c["Hkv"], c["Lq"], c["Lk"]
    scale = c["D"] ** -0.5
    q, k, v = _heads(s["q"], Hkv), _heads(s["k"], Hkv), _heads(s["v"], Hkv)
    allowed = None
    if s["lens"] is not None:
        allowed = torch.arange(Lk, device="cuda") < s["lens"][:, None]
    if s["mask"] is not None:
        allowed = s["mask"] if allowed is None else allowed & s["mask"]
    if allowed is not None:
        k, v = (torch.where(allowed[:, None, :, None], x, 0.0) for x in (k, v))
        allowed = allowed[:, None, None]
    p = _softmax((q * scale) @ k.transpose(-1, -2), allowed)
    o = _tokens(p @ v, Lq, H).to(dt).contiguous()
    if not c["train"]:
        return {"o": o}
    do = _heads(s["do"], Hkv)
    dv = _tokens(p.transpose(-1, -2) @ do, Lk, Hkv).to(dt)
    dp = do @ v.transpose(-1, -2)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    dq = _tokens(ds @ k, Lq, H) * scale
    dk = _tokens(ds.transpose(-1, -2) @ q, Lk, Hkv) * scale
    return {"o": o, "dq": dq.to(dt).contiguous(), "dk": dk.to(dt).contiguous(), "dv": dv.contiguous()}


def _write_plain(s, x):
    """The new tokens of s[x] go into the cache's blocks (the complete ones) and its tail (the last, incomplete one)."""
    new, c8, cs, tail = s[x], s[x + "8"], s[x + "s"], s[x + "t"]
    B, n, Hkv, D = new.shape
    T, block = c8.shape[2], tail.shape[2]
    tail = tail.transpose(1, 2)
    start, total = s["start"].long()[:, None], s["total"].long()[:, None]
    # the blocks that new tokens fall into, complete with the tail's tokens before them
    nb = (n + block - 1) // block + (0 if n % block == 0 and s["case"]["op"] == "fill" else 1)
    at = start // block * block + torch.arange(nb * block, device="cuda")  # (B, nb * block) token of each place
    batch = torch.arange(B, device="cuda")[:, None]
    fresh = new[batch, (at - start).clamp(0, n - 1)]
    held = tail[batch, at % block]
    val = torch.where((at >= start)[..., None, None], fresh, held).float()
    blocks = val.view(B, nb, block, Hkv, D)
    amax = blocks.abs().amax((2, 4))
    scale = amax / torch.full_like(amax, 127.0)
    q = torch.where(scale > 0, scale, 1.0)[:, :, None, :, None]
    eight = torch.round(blocks / q).to(torch.int8)
    which = at[:, ::block] // block  # (B, nb)
    done = (which + 1) * block <= total
    b, j = done.nonzero(as_tuple=True)
    c8.view(B, Hkv, T // block, block, D).permute(0, 2, 3, 1, 4)[b, which[b, j]] = eight[b, j]
    cs.transpose(1, 2)[b, which[b, j]] = scale[b, j]
    b, j = ((at >= start) & (at < total) & (at >= total // block * block)).nonzero(as_tuple=True)
    tail[b, at[b, j] % block] = val[b, j].to(tail.dtype)


def _read_plain(s, x):
    """The cached states in fp32 (B, Hkv, T, D), zero past each sequence's length, and which are there."""
    c8, cs, tail = s[x + "8"], s[x + "s"], s[x + "t"]
    T, block = c8.shape[2], tail.shape[2]
    at, total = torch.arange(T, device="cuda"), s["total"][:, None]
    full = c8.float() * cs.repeat_interleave(block, 2)[..., None]
    full = torch.where((at < total // block * block)[:, None, :, None], full, tail.float()[:, :, at % block])
    return torch.where((at < total)[:, None, :, None], full, 0.0), at < total


@torch.no_grad()
def _kv8_plain(s):
    c = s["case"]
    _write_plain(s, "k")
    _write_plain(s, "v")
    k, there = _read_plain(s, "k")
    v, _ = _read_plain(s, "v")
    dt = s["kt"].dtype
    if c["op"] == "fill":
        return {"k": k.transpose(1, 2).to(dt).contiguous(), "v": v.transpose(1, 2).to(dt).contiguous(), "kt": s["kt"], "vt": s["vt"]}
    q = _heads(s["q"], c["Hkv"])
    p = _softmax((q * c["D"] ** -0.5) @ k.transpose(-1, -2), there[:, None, None])
    return {"o": _tokens(p @ v, c["n"], c["H"]).to(dt).contiguous(), "kt": s["kt"], "vt": s["vt"]}


# ---- what a pass cannot do without --------------------------------------------------------------------
def work(case):
    B, H, Hkv, D = case["B"], case["H"], case["Hkv"], case["D"]
    e = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "rope":
        n = B * (case["Lq"] * H + case["Lk"] * Hkv) * D
        return {"bytes": n * e * (4 if case["train"] else 2), "flops": n * (20 if case["train"] else 6)}
    if case["op"] == "xattn":
        # ragged lengths are spread over [Lk / 2, Lk], and a masked state is no work
        keys = case["Lk"] * (0.75 if case["ragged"] else 1.0) * (0.9 if case["mask"] else 1.0)
        nq, nk = B * case["Lq"] * H * D, B * keys * Hkv * D
        flops = 4.0 * B * H * case["Lq"] * keys * D
        if case["train"]:  # once q, k, v, do in and o, dq, dk, dv out; 2 products forward, 5 backward
            return {"bytes": e * (4 * nq + 4 * nk), "flops": 3.5 * flops}
        return {"bytes": e * (2 * nq + 2 * nk), "flops": flops}
    tokens = 0.75 * case["T"]
    if case["op"] == "fill":
        n = B * tokens * Hkv * D * 2
        return {"bytes": n * (e + 1 + e), "flops": 4 * n}
    n = B * tokens * Hkv * D * 2
    return {"bytes": n + n / D / case["block"] * 4 + e * 2 * B * case["n"] * (H + Hkv) * D,
            "flops": 4.0 * B * case["n"] * H * tokens * D}


# ---- the definition in 64 bits ------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    with torch.enable_grad():
        if case["op"] == "rope":
            return _rope_exact(s)
        if case["op"] == "xattn":
            return _xattn_exact(s)
    return _kv8_exact(s)


def _rope_exact(s):
    """Norm, then each pair of dims as a complex number times exp(i angle); gradients by autograd."""
    c, out = s["case"], {}
    turn = torch.complex(s["cos"].double(), s["sin"].double())
    for n in ("q", "k"):
        x = s[n].detach().double().requires_grad_()
        w = None if s[n + "w"] is None else s[n + "w"].detach().double().requires_grad_()
        y = x / (x.square().sum(-1, keepdim=True) / c["D"] + 1e-6).sqrt()
        if w is not None:
            y = y * w
        head, rest = y.split([c["R"], c["D"] - c["R"]], -1)
        pairs = head.unflatten(-1, (-1, 2)) if c["inter"] else head.unflatten(-1, (2, -1)).transpose(-1, -2)
        z = torch.view_as_complex(pairs.contiguous()) * turn[s[n + "_pos"].long()][:, :, None]
        z = torch.view_as_real(z)
        y = torch.cat(((z if c["inter"] else z.transpose(-1, -2)).flatten(-2), rest), -1)
        out[n] = y.detach()
        if c["train"]:
            grads = torch.autograd.grad(y, (x,) if w is None else (x, w), s["d" + n].double())
            out["d" + n] = grads[0]
            if w is not None:
                out["d" + n + "w"] = grads[1]
    return out


def _xattn_exact(s):
    """One video at a time, over its allowed keys alone; gradients by autograd."""
    c = s["case"]
    G = c["H"] // c["Hkv"]
    outs = {n: [] for n in (("o", "dq", "dk", "dv") if c["train"] else ("o",))}
    for b in range(c["B"]):
        keep = torch.ones(c["Lk"], dtype=torch.bool, device="cuda")
        if s["lens"] is not None:
            keep[int(s["lens"][b]):] = False
        if s["mask"] is not None:
            keep &= s["mask"][b]
        q, k, v = (s[n][b].detach().double().requires_grad_(c["train"]) for n in ("q", "k", "v"))
        kk, vv = (x[keep].repeat_interleave(G, 1).permute(1, 0, 2) for x in (k, v))
        a = torch.softmax(torch.bmm(q.permute(1, 0, 2), kk.mT) / math.sqrt(c["D"]), -1)
        o = torch.bmm(a, vv).permute(1, 0, 2)
        outs["o"].append(o.detach())
        if c["train"]:
            for n, gr in zip(("dq", "dk", "dv"), torch.autograd.grad(o, (q, k, v), s["do"][b].double())):
                outs[n].append(gr)
    return {n: torch.stack(v) for n, v in outs.items()}


@torch.no_grad()
def _kv8_exact(s):
    """The cache's sequences one at a time, on what the 8-bit values stand for."""
    c = s["case"]
    B, T, n, block, G = c["B"], c["T"], c["n"], c["block"], c["H"] // c["Hkv"]
    outs = {x: [] for x in ("k", "v", "o")}
    tails = {x: s[x + "t"].double() for x in ("k", "v")}
    for b in range(B):
        st, total = int(s["start"][b]), int(s["total"][b])
        full, old = total // block, st // block
        vals = {}
        for x in ("k", "v"):
            val = torch.zeros(T, c["Hkv"], c["D"], dtype=torch.float64, device="cuda")
            held = s[x + "8"][b, :, :old * block].transpose(0, 1).double().unflatten(0, (-1, block))
            val[:old * block] = (held * s[x + "s"][b, :, :old].T.double()[:, None, :, None]).flatten(0, 1)
            val[old * block:st] = s[x + "t"][b, :, :st - old * block].transpose(0, 1).double()
            val[st:total] = s[x][b, :total - st].double()
            if full > old:
                blk = val[old * block:full * block].unflatten(0, (-1, block))
                # the scale is an fp32 number by definition, and so is the quotient that is rounded
                sc = blk.abs().amax((1, 3), keepdim=True).float() / torch.tensor(127.0, device="cuda")
                r = torch.round(blk.float() / torch.where(sc > 0, sc, torch.ones_like(sc)))
                val[old * block:full * block] = (r.double() * sc.double()).flatten(0, 1)
            if total > full * block:
                a = max(st, full * block)
                tails[x][b, :, a - full * block:total - full * block] = s[x][b, a - st:total - st].double().transpose(0, 1)
            vals[x] = val
        if c["op"] == "fill":
            outs["k"].append(vals["k"])
            outs["v"].append(vals["v"])
            continue
        kk, vv = (vals[x][:total].repeat_interleave(G, 1).permute(1, 0, 2) for x in ("k", "v"))
        a = torch.softmax(torch.bmm(s["q"][b].double().permute(1, 0, 2), kk.mT) / math.sqrt(c["D"]), -1)
        outs["o"].append(torch.bmm(a, vv).permute(1, 0, 2))
    got = {n: torch.stack(v) for n, v in outs.items() if v}
    return {**got, "kt": tails["k"], "vt": tails["v"]}
