"""What the tests of the paged cache share: caches whose unused places hold NaN, and attention, the 8-bit rows and the
norm computed in 64 bits from their definitions."""
import math

import torch

E4M3 = torch.float8_e4m3fn


def quantise64(x):
    """(e4m3 bytes as float64 values, exponent) of rows, from the definition, on the CPU in 64 bits."""
    x = x.detach().cpu().double()
    mag = torch.where(torch.isnan(x), torch.zeros_like(x), x.abs())
    top = mag.amax(-1) if x.shape[-1] else torch.zeros(x.shape[:-1], dtype=torch.float64)
    e = torch.ceil(torch.log2(top.clamp(1e-300, 1e300) / 448.0)).clamp(-15, 7)
    e = torch.where(top == 0, torch.zeros_like(e), e)
    y = x / torch.pow(2.0, e).unsqueeze(-1)
    y = y.clamp(-448.0, 448.0)                      # (clamp keeps NaN)
    # the nearest multiple of e4m3's step at that magnitude, ties to even; subnormals have steps of 2^-9
    step = torch.pow(2.0, torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
    step = torch.where(torch.isnan(y), torch.ones_like(step), step)
    return torch.round(y / step) * step, e          # torch.round rounds halves to even


def values(cache, exps):
    v = cache.cpu().float().double()
    return v if exps is None else v * torch.pow(2.0, exps.cpu().double() - 127).unsqueeze(-1)


class Cache:
    """A paged cache filled through the plain definition: sequence b holds kv_lens[b] positions; everything else is NaN."""

    def __init__(self, kv_lens, Hkv, D, page, dtype, cache8, seed=0, dev="cuda:0", order="phd", spare=2, scale=1.0):
        g = torch.Generator().manual_seed(seed)
        need = [-(-n // page) for n in kv_lens]
        self.pages, self.page, self.Hkv, self.D = sum(need) + spare, page, Hkv, D
        perm = torch.randperm(self.pages, generator=g).tolist()
        P = max(need + [1])
        self.table = torch.full((len(kv_lens), P), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = torch.tensor(perm[at:at + n], dtype=torch.int32)
            at += n
        self.dense, self.cache, self.exps = [], [], []
        for _ in range(2):
            pool = torch.full((self.pages, Hkv, page, D), float("nan"), dtype=torch.float32)
            ex = torch.full((self.pages, Hkv, page), 255, dtype=torch.uint8) if cache8 else None
            rows = []
            for b, n in enumerate(kv_lens):
                x = (torch.randn(n, Hkv, D, generator=g) * scale).to(dtype)
                pos = torch.arange(n)
                where, off = self.table[b].long()[pos // page], pos % page
                if cache8:
                    q, e = quantise64(x)
                    pool[where, :, off] = q.float()
                    ex[where, :, off] = (e + 127).to(torch.uint8)
                    rows.append(q * torch.pow(2.0, e).unsqueeze(-1))
                else:
                    pool[where, :, off] = x.float()
                    rows.append(x.double())
            pool = pool.to(E4M3 if cache8 else dtype)
            if order == "pdh":        # [pages, page, heads, D] in memory, seen as [pages, heads, page, D]
                raw = pool.view(torch.uint8) if cache8 else pool
                raw = raw.transpose(1, 2).contiguous().to(dev).transpose(1, 2)
                pool = raw.view(E4M3) if cache8 else raw
                ex = ex.transpose(1, 2).contiguous().to(dev).transpose(1, 2) if cache8 else None
            self.cache.append(pool.to(dev))
            self.exps.append(None if ex is None else ex.to(dev))
            self.dense.append(rows)
        self.table = self.table.to(dev)
        self.kv_lens = torch.tensor(kv_lens, dtype=torch.int32, device=dev)

    @property
    def kw(self):
        return {} if self.exps[0] is None else {"k_exp": self.exps[0], "v_exp": self.exps[1]}


def cu_of(lens, first=0, dev="cuda:0"):
    return torch.tensor([first + sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=dev)


def attend64(q, cache, q_lens, kv_lens, scale, causal=True, first=0, absent=()):
    """[(row, head) outputs, lse, tolerance unit] in 64 bits: out, lse, and what one half step of P and of the fp32
    arithmetic may move: A = sum p|v| per element and S = the largest sum |q k| * scale of a row."""
    T, H, D = q.shape
    out, lse = torch.zeros(T, H, D, dtype=torch.float64), torch.full((T, H), -math.inf, dtype=torch.float64)
    A, S = torch.zeros(T, H, D, dtype=torch.float64), torch.zeros(T, H, 1, dtype=torch.float64)
    q = q.detach().cpu().double()
    g = H // cache.Hkv
    t = first
    for b, (n, L) in enumerate(zip(q_lens, kv_lens)):
        gone = torch.zeros(L, dtype=torch.bool)
        for (bb, p) in absent:
            if bb == b:
                gone[p * cache.page:(p + 1) * cache.page] = True
        pos = L - n + torch.arange(n)
        see = (torch.arange(L)[None] <= pos[:, None]) if causal else torch.ones(n, L, dtype=torch.bool)
        see = see & ~gone[None]
        for h in range(H):
            k, v = cache.dense[0][b][:, h // g].clone(), cache.dense[1][b][:, h // g].clone()
            k[gone], v[gone] = 0, 0
            x = (q[t:t + n, h] @ k.T * scale).masked_fill(~see, -math.inf)
            any_ = see.any(1)
            m = x.amax(1, keepdim=True) if L else torch.full((n, 1), -math.inf, dtype=torch.float64)
            m = torch.where(any_[:, None], m, torch.zeros_like(m))
            e = torch.exp(x - m)
            s = e.sum(1, keepdim=True)
            p = torch.where(any_[:, None], e / s.clamp_min(1e-300), torch.zeros_like(e))
            out[t:t + n, h] = p @ v
            lse[t:t + n, h] = torch.where(any_, (m + torch.log(s.clamp_min(1e-300)))[:, 0], torch.full((n,), -math.inf, dtype=torch.float64))
            A[t:t + n, h] = p @ v.abs()
            if L and n:
                # sum |q||k| bounds the fp32 accumulation; max|q| sum|k| what bringing q to another 16-bit type may move
                S[t:t + n, h, 0] = ((q[t:t + n, h].abs() @ k.abs().T) + q[t:t + n, h].abs().amax(1, keepdim=True) * k.abs().sum(1)[None]
                                    ).masked_fill(~see, 0).amax(1) * abs(scale)
        t += n
    return out, lse, A, S


def attend_tolerance(out, A, S, dtype, D, n):
    """Half a step for the output, half a step for each p that multiplies v (16-bit types), and the fp32 arithmetic: a
    score is off by at most (D + 4) half steps of its sum of magnitudes, an exponential by that and 2^-20, a sum of n
    terms by n / 4 + 64 half steps (the kernels sum at least four lanes apart); numerator and denominator both."""
    u, f = torch.finfo(dtype).eps / 2, 2.0 ** -24
    p = u if dtype != torch.float32 else 0.0
    rel = 2 * ((D + 4) * f * S + 2.0 ** -20 + (n / 4 + 64) * f)
    return u * out.abs() + (p * (1 + u) + rel) * A + torch.finfo(dtype).tiny


def lse_tolerance(lse, S, D, n):
    f = 2.0 ** -24
    return (D + 4) * f * S[..., 0] + 2.0 ** -20 + (n / 4 + 64) * f + 4 * f * lse.abs().nan_to_num(posinf=0, neginf=0)
