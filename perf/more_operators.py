"""Workloads of the operators that remember a history: decaying linear attention, a paged 4-bit state cache, its page tables.

``listed()`` names the measured cases, ``draw(rng)`` gives further ones of the
same ranges, ``prepare`` makes what a caller has in hand, ``run`` is one pass.
With ``own`` false the pass is the plain form (elementary torch operations in
fp32, rounded once at the end); with ``own`` true it is the call a user makes
of hclsm_b200.  ``exact`` is the definition in 64 bits.
"""
import math

import torch

own = False

F32, F64, I32, I64 = torch.float32, torch.float64, torch.int32, torch.int64
GROUP = 32  # dims of a head that share one scale of the 4-bit cache


# ---- the cases ----------------------------------------------------------------------------------
def _decay(name, B, L, H, D, *, Dv=0, dtype="bf16", train=True, ragged=False, state=False):
    return {"name": name, "op": "decay", "B": B, "L": L, "H": H, "D": D, "Dv": Dv or D, "dtype": dtype, "train": train,
            "ragged": ragged, "state": state}


def _step(name, B, H, D, *, Dv=0, dtype="bf16"):
    return {"name": name, "op": "step", "B": B, "H": H, "D": D, "Dv": Dv or D, "dtype": dtype}


def _kv4(name, op, B, T, n, H, Hkv, D, *, page=32, dtype="bf16"):
    return {"name": name, "op": op, "B": B, "T": T, "n": n, "H": H, "Hkv": Hkv, "D": D, "page": page, "dtype": dtype}


def _pages(name, B, T, n, *, page=32):
    return {"name": name, "op": "pages", "B": B, "T": T, "n": n, "page": page}


def listed():
    return [
        # an fp32 module over odd, ragged histories that go on from a state (training)
        _decay("decay_odd_train_f32", 3, 333, 6, 64, dtype="f32", ragged=True, state=True),
        # Level-1 widths (d 384 as 6 heads of 64): the 64 x 32 states of 8 videos, a training step
        _decay("decay_events_train", 8, 2048, 6, 64),
        # base width (d 2048 as 16 heads of 128), 16 videos, a training step
        _decay("decay_base_train", 16, 2048, 16, 128),
        # prompts: histories of unequal lengths read without gradients, their states kept
        _decay("decay_prompt", 8, 1000, 32, 64, train=False, ragged=True, state=True),
        # one long history of a single video
        _decay("decay_prompt_long", 1, 65536, 6, 64, train=False, state=True),
        # a rollout step of 8 videos: one token a head through the state
        _step("decay_step", 8, 6, 64),
        # a rollout step of 256 videos at base width
        _step("decay_step_base", 256, 16, 128),
        # the encoder's states of 8 videos written into the paged cache and read back
        _kv4("cache4_fill", "fill", 8, 2048, 2048, 6, 6, 64),
        # a rollout step: one state appended to the cache, one query over it
        _kv4("cache4_step", "attend", 8, 2048, 1, 6, 6, 64),
        # the same over a long history at base width, shared key heads
        _kv4("cache4_step_long", "attend", 16, 65536, 1, 32, 8, 128),
        # a rollout step's pages: 64 videos take one more state each
        _pages("pages_step", 64, 2048, 1),
        # the pages of 64 whole histories
        _pages("pages_prompt", 64, 65536, 65536),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(c):
    """What the plain form goes through, as a share of the largest listed case of the same kind."""
    if c["op"] == "decay":
        n = c["B"] * c["H"] * (c["L"] + 128) * (c["D"] + 128) * (c["Dv"] + 128) * (3 if c["train"] else 1)
        return n / (16 * 16 * 2176 * 256 * 256 * 3)
    if c["op"] == "step":
        return c["B"] * c["H"] * c["D"] * c["Dv"] / (256 * 16 * 128 * 128)
    if c["op"] == "pages":
        return c["B"] * c["T"] / (64 * 65536)
    return c["B"] * c["T"] * c["Hkv"] * c["D"] / (16 * 65536 * 8 * 128)


def draw(rng):
    while True:
        dtype = "f32" if rng.random() < 0.25 else "bf16"
        B, H = _log(rng, 1, 64), _log(rng, 1, 32)
        op = rng.choice(["decay", "decay", "decay", "step", "fill", "attend", "attend", "pages"])
        if op == "decay":
            D = rng.choice([32, 64, 64, 96, 128])
            c = _decay("", B, _log(rng, 1, 16384), H, D, Dv=rng.choice([D, D, 32, 64, 128]), dtype=dtype,
                       train=rng.random() < 0.6, ragged=rng.random() < 0.5, state=rng.random() < 0.5)
            if dtype == "f32" and _cost(c) > 0.25:
                continue
        elif op == "step":
            D = rng.choice([32, 64, 96, 128])
            c = _step("", _log(rng, 1, 512), H, D, Dv=rng.choice([D, D, 64, 128]), dtype=dtype)
        elif op == "pages":
            page, T = rng.choice([16, 32, 64, 128]), _log(rng, 64, 65536)
            c = _pages("", _log(rng, 1, 512), T, rng.choice([1, 1, _log(rng, 1, T)]), page=page)
        else:
            G, Hkv, page = rng.choice([1, 1, 2, 4, 5, 8]), _log(rng, 1, 12), rng.choice([16, 32, 64, 128])
            T = max(1, _log(rng, 64, 65536 if op == "attend" else 4096) // page) * page
            n = T if op == "fill" else rng.choice([1, 1, 1, 7, 32])
            c = _kv4("", op, B, T, n, Hkv * G, Hkv, rng.choice([32, 64, 96, 128]), page=page, dtype=dtype)
            if op == "fill":
                c["H"] = Hkv
            elif _cost(c) * n * G > 4 or B * c["H"] * n * T > 1 << 30:
                continue
        if _cost(c) <= 1 and (op != "fill" or _cost(c) <= 0.1):
            del c["name"]
            return c


# ---- inputs ---------------------------------------------------------------------------------------
def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else F32


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    B, s = case["B"], {"case": case}

    def randn(*shape, dt=None):
        return torch.randn(*shape, generator=g, device="cuda", dtype=F32).to(dt or _dtype(case))

    def ints(lo, hi, *shape, dt=I32):
        return torch.randint(lo, hi, shape, generator=g, device="cuda", dtype=dt)

    if case["op"] == "pages":
        T, n, page = case["T"], case["n"], case["page"]
        M = (T + page - 1) // page
        new = ints(max(T // 2, n), T + 1, B)
        s["old"], s["new"] = (new - n).contiguous(), new
        # every entry's pages lie scattered over the pool, which holds a tenth more than all could take
        P = B * M + B * M // 10 + 1
        order = torch.randperm(P, generator=g, device="cuda").to(I32)
        table = order[:B * M].view(B, M)
        held = torch.arange(M, device="cuda") < ((s["old"] + page - 1) // page)[:, None]
        s["table"] = torch.where(held, table, -1).contiguous()
        free = torch.cat((order[B * M:], table[~held]))
        s["free"] = torch.cat((free, free.new_full((P - free.numel(),), -1)))
        s["n_free"] = torch.tensor([free.numel()], device="cuda", dtype=I32)
        return s
    H, D = case["H"], case["D"]
    if case["op"] in ("decay", "step"):
        Dv = case["Dv"]
        L = () if case["op"] == "step" else (case["L"],)
        # keys of norm one, as after a norm of the heads; heads forget over some 4 to 4000 tokens
        s["q"], s["k"], s["v"] = randn(B, *L, H, D), (randn(B, *L, H, D, dt=F32) * D ** -0.5).to(_dtype(case)), randn(
            B, *L, H, Dv)
        s["decay"] = torch.log1p(-(2.0 ** -torch.linspace(2, 12, H, device="cuda", dtype=F64))).float()
        s["state"] = randn(B, H, D, Dv, dt=F32) if L == () or case["state"] else None
        if L == ():
            s["next"] = torch.empty(B, H, D, Dv, device="cuda")
            return s
        s["lens"] = ints(L[0] // 2, L[0] + 1, B) if case["ragged"] else None
        if case["train"]:
            s["do"] = randn(B, *L, H, Dv)
            s["ds"] = randn(B, H, D, Dv, dt=F32) if case["state"] else None
            for n in ("q", "k", "v", "state"):
                if s[n] is not None:
                    s[n].requires_grad_()
        return s
    T, n, page, Hkv = case["T"], case["n"], case["page"], case["Hkv"]
    M = T // page
    P = B * M + 8
    s["table"] = torch.randperm(P, generator=g, device="cuda").to(I32)[:B * M].view(B, M).contiguous()
    s["k"], s["v"] = randn(B, n, Hkv, D), randn(B, n, Hkv, D)
    for x in ("k", "v"):
        if case["op"] == "fill":
            s[x + "4"] = torch.zeros(P, Hkv, page, D // 2, dtype=torch.uint8, device="cuda")
            s[x + "s"] = torch.zeros(P, Hkv, page, D // GROUP, dtype=torch.bfloat16, device="cuda")
        else:
            s[x + "4"] = ints(0, 256, P, Hkv, page, D // 2, dt=torch.uint8)
            s[x + "s"] = (torch.rand(P, Hkv, page, D // GROUP, generator=g, device="cuda") * 0.1 + 0.2).to(torch.bfloat16)
    if case["op"] == "fill":
        s["start"] = torch.zeros(B, dtype=I32, device="cuda")
        s["count"] = ints(n // 2, n + 1, B)
    else:
        s["q"] = randn(B, n, H, D)
        s["start"] = ints(max(T // 2 - n, 0), T - n + 1, B)
        s["count"] = torch.full((B,), n, dtype=I32, device="cuda")
    s["total"] = s["start"] + s["count"]
    return s


# ---- one pass ---------------------------------------------------------------------------------------
def run(s):
    op = s["case"]["op"]
    if op == "decay":
        return _decay_own(s) if own else _decay_plain(s)
    if op == "step":
        return _step_own(s) if own else _step_plain(s)
    if op == "pages":
        return _pages_own(s) if own else _pages_plain(s)
    return _kv4_own(s) if own else _kv4_plain(s)


def _decay_own(s):
    from hclsm_b200.kernels import decay_attention

    o, state = decay_attention(s["q"], s["k"], s["v"], s["decay"], state=s["state"], lens=s["lens"], return_state=True)
    if not s["case"]["train"]:
        return {"o": o, "state": state}
    names = [n for n in ("q", "k", "v", "state") if s[n] is not None]
    out, up = ((o,), (s["do"],)) if s["ds"] is None else ((o, state), (s["do"], s["ds"]))
    grads = torch.autograd.grad(out, [s[n] for n in names], up)
    return {"o": o.detach(), "state": state.detach(), **{"d" + n: g for n, g in zip(names, grads)}}


def _step_own(s):
    from hclsm_b200.kernels import decay_attention_step

    return {"o": decay_attention_step(s["q"], s["k"], s["v"], s["decay"], s["state"], out=s["next"]), "state": s["next"]}


def _kv4_own(s):
    from hclsm_b200.kernels import Kv4Cache, kv4_attention, kv4_read, kv4_write, page_slots

    cache = Kv4Cache(s["k4"], s["v4"], s["ks"], s["vs"], _dtype(s["case"]))
    slots = page_slots(s["table"], s["start"], s["case"]["n"], count=s["count"], page=s["case"]["page"])
    kv4_write(cache, s["k"], s["v"], slots)
    if s["case"]["op"] == "fill":
        k, v = kv4_read(cache, s["table"], s["total"])
        return {"k": k, "v": v}
    return {"o": kv4_attention(s["q"], cache, s["table"], s["total"]), "slots": slots, "ks": s["ks"], "vs": s["vs"]}


def _pages_own(s):
    from hclsm_b200.kernels import PageTable, page_slots, pages_resize

    c = s["case"]
    pages = PageTable(s["table"], s["free"], s["n_free"], c["page"])
    pages_resize(pages, s["old"], s["new"])
    slots = page_slots(pages.table, s["old"], c["n"], page=c["page"])
    left = s["n_free"].clone()
    pages_resize(pages, s["new"], s["old"])  # the branch is given up: as before
    return {"slots": slots, "left": left, "table": s["table"], "free": s["free"], "n_free": s["n_free"]}


def _valid(s):
    """(B, L) whether a token counts."""
    L = s["case"]["L"]
    n = torch.full((s["case"]["B"],), L, device="cuda") if s["lens"] is None else s["lens"]
    return torch.arange(L, device="cuda") < n[:, None], n


def _chunked(q, k, v, g, S0, C):
    """o_t = q_t (g^(t + 1) S0 + sum over s <= t of g^(t - s) k_s^T v_s) for q, k (B, H, n, C, D), v (B, H, n, C, Dv) by
    chunks of C tokens; g (H,) the logarithms of the decays."""
    n, H = q.shape[2], g.shape[0]
    at = torch.arange(C, device="cuda")
    lag = (at[:, None] - at).double()
    w = torch.where(lag >= 0, torch.exp(g.double()[:, None, None] * lag.clamp(min=0)), 0.0).float()
    o = ((q @ k.transpose(-1, -2)) * w[:, None]) @ v
    # the states before each chunk: the chunks' sums, weighted by how many chunks ago they were
    rest = torch.exp(g.double()[:, None] * (C - 1 - at).double()).float()
    sums = (k * rest[:, None, :, None]).transpose(-1, -2) @ v
    ago = (torch.arange(n, device="cuda")[:, None] - 1 - torch.arange(n, device="cuda")).double()
    w = torch.where(ago >= 0, torch.exp(g.double()[:, None, None] * C * ago.clamp(min=0)), 0.0).float()
    before = (w @ sums.flatten(3)).view_as(sums)
    if S0 is not None:
        first = torch.exp(g.double()[:, None] * C * torch.arange(n, device="cuda")).float()
        before += first[:, :, None, None] * S0[:, :, None]
    lead = torch.exp(g.double()[:, None] * (at + 1)).float().view(H, 1, C, 1)
    return o + lead * (q @ before)


@torch.no_grad()
def _decay_plain(s):
    c, g, dt = s["case"], s["decay"], s["q"].dtype
    B, L, H = c["B"], c["L"], c["H"]
    C = min(128, L)
    pad = -L % C
    there, n = _valid(s)

    def chunks(x):
        x = torch.where(there[:, :, None, None], x.float(), 0.0)
        x = torch.nn.functional.pad(x, (0, 0, 0, 0, 0, pad))
        return x.permute(0, 2, 1, 3).reshape(B, H, -1, C, x.shape[-1])

    def back(x):
        x = x.reshape(B, H, L + pad, -1)[:, :, :L].permute(0, 2, 1, 3)
        return torch.where(there[:, :, None, None], x, 0.0).to(dt).contiguous()

    scale = c["D"] ** -0.5
    q, k, v, S0 = chunks(s["q"]) * scale, chunks(s["k"]), chunks(s["v"]), s["state"]
    out = {"o": back(_chunked(q, k, v, g, S0, C))}
    at, n = torch.arange(L + pad, device="cuda"), n[:, None]
    # the state behind token n - 1, n each entry's length
    lag = (n - 1 - at).double()[:, None]
    w = torch.where(lag >= 0, torch.exp(g.double()[:, None] * lag.clamp(min=0)), 0.0).float()[..., None]
    state = (k.flatten(2, 3) * w).transpose(-1, -2) @ v.flatten(2, 3)
    all_of = torch.exp(g.double() * n).float()[..., None, None]
    out["state"] = state if S0 is None else state + all_of * S0
    if not c["train"]:
        return out
    do = chunks(s["do"])
    ds = s["ds"]
    # dq looks back over v and k; dv and dk look ahead, which is looking back in reversed order, where the
    # gradient of the state behind the last token enters each token by its distance from it
    dq = _chunked(do, v, k, g, None if S0 is None else S0.transpose(-1, -2), C)
    rq, rk, rv, rdo = (x.flatten(2, 3).flip(2).view_as(x) for x in (q, k, v, do))
    dv = _chunked(rk, rq, rdo, g, None, C).flatten(2, 3).flip(2)
    dk = _chunked(rv, rdo, rq, g, None, C).flatten(2, 3).flip(2)
    if ds is not None:
        dv += w * (k.flatten(2, 3) @ ds)
        dk += w * (v.flatten(2, 3) @ ds.transpose(-1, -2))
    out.update(dq=back(dq * scale), dk=back(dk), dv=back(dv))
    if S0 is not None:
        lead = torch.exp(g.double()[:, None] * (at + 1)).float()[..., None]
        out["dstate"] = (q.flatten(2, 3) * lead).transpose(-1, -2) @ do.flatten(2, 3)
        if ds is not None:
            out["dstate"] += all_of * ds
    return out


@torch.no_grad()
def _step_plain(s):
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    S = torch.exp(s["decay"])[:, None, None] * s["state"] + k[..., None] * v[..., None, :]
    o = (q[..., None, :] @ S)[..., 0, :] * s["case"]["D"] ** -0.5
    s["next"].copy_(S)
    return {"o": o.to(s["q"].dtype), "state": s["next"]}


def _slots_plain(table, start, n, count, page):
    """(B, n) the pool's slot of tokens start, start + 1, ... of each entry; -1 behind its count."""
    at = start[:, None] + torch.arange(n, device="cuda", dtype=I32)
    there = at < (start + count)[:, None]
    got = table.gather(1, (at // page).clamp(max=table.shape[1] - 1).long())
    return torch.where(there & (got >= 0), got * page + at % page, -1)


def _codes(x):
    """(codes 0 to 15, scales) of x (..., D): groups of 32 dims, scale = the value of largest magnitude / -8 as bf16
    (the positive one where both signs have it), code = the nearest whole number of x / scale in [-8, 7], plus 8."""
    x = x.float().unflatten(-1, (-1, GROUP))
    hi, lo = x.amax(-1), x.amin(-1)
    top = torch.where(hi >= -lo, hi, lo)
    scale = (top / -8.0).to(torch.bfloat16)
    # the quotient in 64 bits: fp32 would put values next to the middle of two codes onto it
    quotient = x.double() / torch.where(scale == 0, 1.0, scale.double())[..., None]
    codes = torch.round(quotient).clamp(-8, 7) + 8
    return torch.where(scale[..., None] == 0, 8.0, codes).to(torch.uint8).flatten(-2), scale


def _order(D):
    """The dims in the order of their 4 bits in memory (the low half of a byte first): runs of four, those of dims d to
    d + 3 and of d + 32 to d + 35 of each 64 beside each other; 32 dims behind the last 64 as they are."""
    at, whole = torch.arange(D, device="cuda"), D // 64 * 64
    return torch.cat((at[:whole].view(-1, 2, 8, 4).transpose(1, 2).flatten(), at[whole:]))


@torch.no_grad()
def _write_plain(s, x, slots):
    new, c4, cs = s[x], s[x + "4"], s[x + "s"]
    page = c4.shape[2]
    codes, scale = _codes(new)
    stored = codes[..., _order(codes.shape[-1])]
    packed = stored[..., 0::2] | stored[..., 1::2] << 4
    b, i = (slots >= 0).nonzero(as_tuple=True)
    at = slots[b, i].long()
    c4[at // page, :, at % page] = packed[b, i]
    cs[at // page, :, at % page] = scale[b, i]


def _read_plain(s, x):
    """The cached states in fp32 (B, Hkv, T, D), zero past each sequence's length, and which are there."""
    c = s["case"]
    c4, cs, table = s[x + "4"], s[x + "s"], s["table"].long()
    bytes_ = c4[table].transpose(1, 2).flatten(2, 3)  # (B, Hkv, T, D / 2)
    stored = torch.stack((bytes_ & 15, bytes_ >> 4), -1).flatten(-2).float() - 8.0
    codes = torch.empty_like(stored)
    codes[..., _order(c["D"])] = stored
    scale = cs[table].transpose(1, 2).flatten(2, 3).float()
    full = (codes.unflatten(-1, (-1, GROUP)) * scale[..., None]).flatten(-2)
    there = torch.arange(c["T"], device="cuda") < s["total"][:, None]
    return torch.where(there[:, None, :, None], full, 0.0), there


@torch.no_grad()
def _kv4_plain(s):
    c = s["case"]
    dt = _dtype(c)
    slots = _slots_plain(s["table"], s["start"], c["n"], s["count"], c["page"])
    _write_plain(s, "k", slots)
    _write_plain(s, "v", slots)
    k, there = _read_plain(s, "k")
    v, _ = _read_plain(s, "v")
    if c["op"] == "fill":
        return {"k": k.transpose(1, 2).to(dt).contiguous(), "v": v.transpose(1, 2).to(dt).contiguous()}
    B, n, H, D, Hkv = c["B"], c["n"], c["H"], c["D"], c["Hkv"]
    q = s["q"].float().permute(0, 2, 1, 3).reshape(B, Hkv, H // Hkv * n, D)
    scores = ((q * D ** -0.5) @ k.transpose(-1, -2)).masked_fill(~there[:, None, None], -torch.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    o = ((p / p.sum(-1, keepdim=True)) @ v).reshape(B, H, n, D).permute(0, 2, 1, 3).to(dt).contiguous()
    return {"o": o, "slots": slots, "ks": s["ks"], "vs": s["vs"]}


def _resize_plain(s, old, new):
    """Entries' pages from those of old tokens to those of new ones: the released ones go onto the free list, the
    first of them last, then the wanted ones come off its end."""
    table, free, page = s["table"], s["free"], s["case"]["page"]
    had, has = (old + page - 1) // page, (new + page - 1) // page
    at = torch.arange(table.shape[1], device="cuda")
    gone = ((at >= has[:, None]) & (at < had[:, None])).flatten()
    want = ((at >= had[:, None]) & (at < has[:, None])).flatten()
    n, flat = s["n_free"].long(), table.view(-1)
    released, wanted = gone.sum(), want.sum()
    which = gone.nonzero()[:, 0]
    free[n + released - 1 - torch.arange(which.numel(), device="cuda")] = flat[which]
    flat[which] = -1
    which = want.nonzero()[:, 0]
    take = n + released - 1 - torch.arange(which.numel(), device="cuda")
    flat[which] = free[take]
    free[take] = -1
    s["n_free"].copy_(n + released - wanted)


@torch.no_grad()
def _pages_plain(s):
    c = s["case"]
    _resize_plain(s, s["old"], s["new"])
    slots = _slots_plain(s["table"], s["old"], c["n"], torch.full_like(s["old"], c["n"]), c["page"])
    left = s["n_free"].clone()
    _resize_plain(s, s["new"], s["old"])
    return {"slots": slots, "left": left, "table": s["table"], "free": s["free"], "n_free": s["n_free"]}


# ---- what a pass cannot do without --------------------------------------------------------------------
def work(case):
    B = case["B"]
    if case["op"] == "pages":
        # the slots written; lengths read, the pages of the grown part popped and put into the table, and back
        moved = B * (case["n"] + case["page"] - 1) // case["page"]
        return {"bytes": 4 * (B * case["n"] + 4 * moved + 6 * B), "flops": 0}
    H, D = case["H"], case["D"]
    e = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "step":
        n = B * H * D * case["Dv"]
        return {"bytes": 8 * n + e * B * H * 2 * (D + case["Dv"]), "flops": 5 * n}
    if case["op"] == "decay":
        Dv = case["Dv"]
        tokens = B * case["L"] * H * (0.75 if case["ragged"] else 1.0)
        io, S = tokens * e, B * H * D * Dv * 4
        states = S * (2 if case["state"] else 1)
        flops = 4.0 * tokens * D * Dv  # the recurrence: a state's update and its reading
        if case["train"]:  # q, k, v, do in and o, dq, dk, dv out
            return {"bytes": io * 4 * (D + Dv) + states * (2 if case["state"] else 1), "flops": 4.0 * flops}
        return {"bytes": io * 2 * (D + Dv) + states, "flops": flops}
    Hkv, tokens = case["Hkv"], 0.75 * case["T"]
    four = B * tokens * Hkv * D * 2 * (0.5 + 2 / GROUP)  # codes and scales of both
    if case["op"] == "fill":
        return {"bytes": four + 2 * e * B * tokens * Hkv * D * 2, "flops": 8 * B * tokens * Hkv * D}
    return {"bytes": four + e * 2 * B * case["n"] * (H + Hkv) * D, "flops": 4.0 * B * case["n"] * H * tokens * D}


# ---- the definition in 64 bits ------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "decay":
        with torch.enable_grad():
            return _decay_exact(s)
    if case["op"] == "step":
        return _step_exact(s)
    if case["op"] == "pages":
        return _pages_exact(s)
    return _kv4_exact(s)


def _decay_exact(s):
    """One entry and some heads at a time, every pair of tokens by its distance, in spans of queries; a span's
    gradients by autograd, summed."""
    c = s["case"]
    B, L, H, D, Dv = c["B"], c["L"], c["H"], c["D"], c["Dv"]
    if B * H * float(L) ** 2 * (D + Dv) * (4 if c["train"] else 1) > 3e13:
        return None
    scale = D ** -0.5
    g = s["decay"].double()
    out = {"o": torch.zeros(B, L, H, Dv, dtype=F64, device="cuda"), "state": torch.zeros(B, H, D, Dv, dtype=F64, device="cuda")}
    if c["train"]:
        for n in ("q", "k", "v", "state"):
            if s[n] is not None:
                out["d" + n] = torch.zeros(s[n].shape, dtype=F64, device="cuda")
    span = 1024
    for b in range(B):
        n = L if s["lens"] is None else int(s["lens"][b])
        for h in range(H):
            q, k, v = (s[x][b, :n, h].detach().double().requires_grad_(c["train"]) for x in ("q", "k", "v"))
            S0 = None if s["state"] is None else s["state"][b, h].detach().double().requires_grad_(c["train"])
            at = torch.arange(n, device="cuda", dtype=F64)
            leaves = [x for x in (q, k, v, S0) if x is not None]
            sums = [torch.zeros_like(x) for x in leaves]

            def add(y, up):
                if c["train"] and up is not None and y.requires_grad:
                    for t, gr in zip(sums, torch.autograd.grad(y, leaves, up.double(), allow_unused=True)):
                        if gr is not None:
                            t += gr

            for i in range(0, n, span):
                lag = at[i:i + span, None] - at[:i + span]
                w = torch.exp(g[h] * lag.clamp(min=0)) * (lag >= 0)
                y = ((q[i:i + span] @ k[:i + span].T) * w) @ v[:i + span]
                if S0 is not None:
                    y = y + torch.exp(g[h] * (at[i:i + span, None] + 1)) * (q[i:i + span] @ S0)
                y = y * scale
                out["o"][b, i:min(i + span, n), h] = y.detach()
                if c["train"]:
                    add(y, s["do"][b, i:min(i + span, n), h])
            S = (k * torch.exp(g[h] * (n - 1 - at))[:, None]).T @ v
            if S0 is not None:
                S = S + torch.exp(g[h] * n) * S0
            out["state"][b, h] = S.detach()
            if c["train"]:
                add(S, None if s["ds"] is None else s["ds"][b, h])
                names = [x for x in ("q", "k", "v", "state") if s[x] is not None]
                for x, t in zip(names, sums):
                    if x == "state":
                        out["dstate"][b, h] = t
                    else:
                        out["d" + x][b, :n, h] = t
    return out


def _step_exact(s):
    S = s["state"].double() * s["decay"].double().exp().view(-1, 1, 1) + torch.einsum("bhi,bhj->bhij", s["k"].double(), s["v"].double())
    return {"o": torch.einsum("bhi,bhij->bhj", s["q"].double(), S) / math.sqrt(s["case"]["D"]), "state": S}


def _pages_exact(s):
    """The same lists on the host, one page at a time."""
    c = s["case"]
    page = c["page"]
    table, free, n = s["table"].cpu().tolist(), s["free"].cpu().tolist(), int(s["n_free"])
    old, new = s["old"].tolist(), s["new"].tolist()
    for b in range(c["B"]):
        for j in range(-(-old[b] // page), -(-new[b] // page)):
            n -= 1
            table[b][j], free[n] = free[n], -1
    left, cols = n, torch.arange(c["n"])
    t = torch.tensor(table)
    at = torch.tensor(old)[:, None] + cols
    slots = torch.gather(t, 1, at // page) * page + at % page
    return {"slots": slots.to(I32).cuda(), "left": torch.tensor([left], dtype=I32, device="cuda"), "table": s["table"],
            "free": s["free"], "n_free": s["n_free"]}


@torch.no_grad()
def _kv4_exact(s):
    """The cache's sequences one at a time, on what the 4-bit values stand for."""
    c = s["case"]
    B, T, n, page, Hkv, D = c["B"], c["T"], c["n"], c["page"], c["Hkv"], c["D"]
    G = c["H"] // Hkv
    outs = {x: [] for x in ("k", "v", "o")}
    state = {} if c["op"] == "fill" else {"slots": torch.empty(B, n, dtype=I32, device="cuda"), "ks": s["ks"].double(),
                                          "vs": s["vs"].double()}
    for b in range(B):
        st, total = int(s["start"][b]), int(s["total"][b])
        ids = s["table"][b].long()
        vals = {}
        for x in ("k", "v"):
            val = torch.zeros(T, Hkv, D, dtype=F64, device="cuda")
            byte = s[x + "4"][ids].permute(0, 2, 1, 3).reshape(T, Hkv, D // 2)[:st].int()
            for d in range(D):  # where dim d's four bits are
                at = d // 64 * 64 + (d % 32 // 4 * 8 + d % 64 // 32 * 4 + d % 4 if d < D // 64 * 64 else d % 64)
                val[:st, :, d] = ((byte[..., at // 2] >> 4 * (at % 2)) % 16 - 8).double()
            sc = s[x + "s"][ids].permute(0, 2, 1, 3).reshape(T, Hkv, D // GROUP)[:st].double()
            val[:st] *= sc.repeat_interleave(GROUP, -1)
            new = s[x][b, :total - st].double().reshape(total - st, Hkv, D // GROUP, GROUP)
            mag = new.abs().amax(-1, keepdim=True)
            sign = torch.where((new == mag).any(-1, keepdim=True), 1.0, -1.0)
            # the scale is a bf16 number by definition
            sc = (mag * sign / -8.0).float().to(torch.bfloat16).double()
            r = torch.where(sc != 0, torch.round(new / torch.where(sc != 0, sc, 1.0)).clamp(-8, 7), 0.0)
            val[st:total] = (r * sc).flatten(-2)
            vals[x] = val
            if state:
                at = torch.arange(st, total, device="cuda")
                state["slots"][b] = ids[at // page] * page + at % page
                state[x + "s"][ids[at // page], :, at % page] = sc[..., 0]
        if c["op"] == "fill":
            outs["k"].append(vals["k"])
            outs["v"].append(vals["v"])
            continue
        kk, vv = (vals[x][:total].permute(1, 0, 2) for x in ("k", "v"))
        q = s["q"][b].double().view(n, Hkv, G, D).permute(1, 2, 0, 3).reshape(Hkv, G * n, D)
        o = torch.softmax(q @ kk.mT / math.sqrt(D), -1) @ vv
        outs["o"].append(o.view(Hkv, G, n, D).permute(2, 0, 1, 3).reshape(n, c["H"], D))
    return {**{x: torch.stack(v) for x, v in outs.items() if v}, **state}
