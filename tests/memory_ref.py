"""Plain definitions in 64 bits of the operators that remember a history (any device), for the tests."""
import torch

F64 = torch.float64


def decay_ref(q, k, v, g, S0=None, lens=None, scale=1.0):
    """(o, final state) by the recurrence's closed form; g (H,) logarithms of the decays."""
    q, k, v, g = q.to(F64), k.to(F64), v.to(F64), g.to(F64)
    B, L, H, D = q.shape
    n = torch.full((B,), L, device=q.device) if lens is None else lens.clamp(0, L).long()
    at = torch.arange(L, device=q.device)
    there = (at < n[:, None])[:, None, :, None]
    q, k, v = (torch.where(there, x.transpose(1, 2), 0.0) for x in (q, k, v))
    lag = at[:, None] - at
    w = torch.where(lag >= 0, torch.exp(g[:, None, None] * lag.clamp(min=0)), 0.0)
    o = ((q @ k.mT) * w) @ v
    last = (n[:, None] - 1 - at).clamp(min=0)  # (B, L)
    S = (k * torch.exp(g[:, None] * last[:, None])[..., None]).mT @ v
    if S0 is not None:
        S0 = S0.to(F64)
        o = o + torch.exp(g[:, None] * (at + 1))[..., None] * (q @ S0)
        S = S + torch.exp(g * n[:, None])[..., None, None] * S0
    return torch.where(there, scale * o, 0.0).transpose(1, 2), S


def decay_grads(q, k, v, g, S0, lens, scale, do, dS):
    """(dq, dk, dv, dS0 or None) by the formulas, written out."""
    q, k, v, g, do = (x.to(F64) for x in (q, k, v, g, do))
    B, L, H, D = q.shape
    n = torch.full((B,), L, device=q.device) if lens is None else lens.clamp(0, L).long()
    at = torch.arange(L, device=q.device)
    there = (at < n[:, None])[:, None, :, None]
    q, k, v, do = (torch.where(there, x.transpose(1, 2), 0.0) for x in (q, k, v, do))
    lag = at[:, None] - at
    w = torch.where(lag >= 0, torch.exp(g[:, None, None] * lag.clamp(min=0)), 0.0)
    a, da = (q @ k.mT) * w, (do @ v.mT) * w
    dq, dk, dv = scale * da @ k, scale * da.mT @ q, scale * a.mT @ do
    lead = torch.exp(g[:, None] * (at + 1))[..., None]
    last = torch.exp(g[:, None] * (n[:, None] - 1 - at).clamp(min=0)[:, None])[..., None]
    dS0 = None
    if S0 is not None:
        dq = dq + scale * lead * (do @ S0.to(F64).mT)
        dS0 = scale * (lead * q).mT @ do
    if dS is not None:
        dS = dS.to(F64)
        dk = dk + last * (v @ dS.mT)
        dv = dv + last * (k @ dS)
        if S0 is not None:
            dS0 = dS0 + torch.exp(g * n[:, None])[..., None, None] * dS
    dq, dk, dv = (torch.where(there, x, 0.0).transpose(1, 2) for x in (dq, dk, dv))
    return dq, dk, dv, dS0


def kv4_ref(x):
    """(codes 0 to 15, scales) of x (..., D): groups of 32, scale = bf16(value of largest magnitude / -8), halves to even."""
    x = x.float().unflatten(-1, (-1, 32))
    hi, lo = x.amax(-1), x.amin(-1)
    top = torch.where(hi >= -lo, hi, lo)
    scale = (top / -8.0).bfloat16()
    r = torch.round(x.double() / torch.where(scale == 0, 1.0, scale.double())[..., None]).clamp(-8, 7) + 8
    return torch.where(scale[..., None] == 0, 8.0, r).flatten(-2).to(torch.uint8), scale


def kv4_values(codes, scale):
    return ((codes.double() - 8).unflatten(-1, (-1, 32)) * scale.double()[..., None]).flatten(-2)


def kv4_unpack(bytes_):
    """Codes (..., D) of packed bytes (..., D / 2), one dim at a time."""
    D = 2 * bytes_.shape[-1]
    out = torch.empty(*bytes_.shape[:-1], D, dtype=torch.uint8, device=bytes_.device)
    for d in range(D):
        block, r = divmod(d, 64)
        at = block * 64 + (r % 32 // 4 * 8 + r // 32 * 4 + r % 4 if block * 64 + 64 <= D else r)
        out[..., d] = bytes_[..., at // 2] >> 4 * (at % 2) & 15
    return out


class PagesRef:
    """The page tables as Python lists."""

    def __init__(self, table, free, n_free, page):
        self.table, self.free, self.page = table.tolist(), free.tolist(), page
        self.n = int(n_free)

    def resize(self, old, new):
        M, P, page = len(self.table[0]) if self.table else 0, len(self.free), self.page
        had, has = ([-(-x // page) for x in y] for y in (old, new))
        if any(not 0 <= x <= M * page for x in old + new) or not 0 <= self.n <= P:
            return False
        gone = [self.table[b][j] for b in range(len(old)) for j in range(has[b], had[b])]
        wanted = sum(max(0, has[b] - had[b]) for b in range(len(old)))
        if self.n + len(gone) > P or wanted > self.n + len(gone) or any(not 0 <= p < P for p in gone):
            return False
        stack = self.free[:self.n] + gone[::-1]
        taken = stack[len(stack) - wanted:][::-1]
        if any(not 0 <= p < P for p in taken):
            return False
        for b in range(len(old)):
            for j in range(has[b], had[b]):
                self.table[b][j] = -1
            for j in range(had[b], has[b]):
                self.table[b][j] = taken.pop(0)
        self.n = len(stack) - wanted
        self.free[:len(stack)] = stack[:self.n] + [-1] * wanted
        return True
