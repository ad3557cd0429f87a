"""What a serving step of a decoder layer does around its projections, and the training form of its norm:

  attend   attention of new tokens (one each, a few drafted ones, or a chunk) over a paged cache
  write    new keys and values put into the paged cache, as they are or in 8 bits
  read     the cache's sequences read back as dense 16-bit rows
  norm     residual addition and RMSNorm: with an 8-bit output and scales, or trained through

`run` computes each in elementary torch operations where `own` is false, and calls the framework where it is true.
Layouts: new tokens are ragged, sequence b has the rows cu_q[b] .. cu_q[b+1]-1 of q / k / v [tokens, heads, D]; caches are
[pages, kv heads, page, D]; page_table[b] names the pages of sequence b; kv_lens[b] counts its positions, the new tokens
(its last ones) among them.  8-bit caches hold e4m3 and one exponent byte e per row: a value is e4m3 * 2^(e - 127).
"""
import math
import os
import random
import sys

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "e4m3": torch.float8_e4m3fn}
SIZES = {"bf16": 2, "fp16": 2, "fp32": 4, "e4m3": 1}
E_LO, E_HI = -15, 7   # exponents of the 8-bit cache: everything it can hold is exact in bf16 and fp16


def _abi():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "framework-torch-paras_b200", "python")
    if root not in sys.path:
        sys.path.insert(0, root)
    from torch_paras import abi
    return abi


# ---------------------------------------------------------------- cases

def listed():
    return [
        # one user's next token over a short chat: latency
        dict(name="attend_token_1x1k", op="attend", type="bf16", cache="bf16", seqs=1, q=1, long_q=0,
             kv_lo=1000, kv_hi=1000, heads=32, kv_heads=8, dim=128, page=16, lens=1),
        # a decode batch of very different cache lengths
        dict(name="attend_token_64x16k", op="attend", type="bf16", cache="bf16", seqs=64, q=1, long_q=0,
             kv_lo=512, kv_hi=16384, heads=32, kv_heads=8, dim=128, page=16, lens=2),
        # four drafted tokens a sequence are checked against an 8-bit cache
        dict(name="attend_draft_48x8k_e4m3", op="attend", type="fp16", cache="e4m3", seqs=48, q=4, long_q=0,
             kv_lo=300, kv_hi=8192, heads=32, kv_heads=8, dim=128, page=64, lens=3),
        # long prompts brought in by chunks of 2048 tokens
        dict(name="attend_chunk_2x2048_8k", op="attend", type="bf16", cache="bf16", seqs=2, q=2048, long_q=0,
             kv_lo=6000, kv_hi=8192, heads=32, kv_heads=8, dim=128, page=64, lens=4),
        # a step that mixes one chunk of a prompt with other users' single tokens, 8-bit cache, groups of three heads
        dict(name="attend_mixed_12x4k_e4m3", op="attend", type="bf16", cache="e4m3", seqs=12, q=1, long_q=700,
             kv_lo=701, kv_hi=4096, heads=24, kv_heads=8, dim=64, page=32, lens=5),
        # a decode step's keys and values into an 8-bit cache: latency
        dict(name="write_token_64_e4m3", op="write", type="bf16", cache="e4m3", seqs=64, q=1, long_q=0,
             kv_lo=10, kv_hi=600, kv_heads=8, dim=128, page=16, lens=6),
        # a prefill step's
        dict(name="write_chunk_4x4096_e4m3", op="write", type="fp16", cache="e4m3", seqs=4, q=4096, long_q=0,
             kv_lo=4096, kv_hi=6000, kv_heads=8, dim=128, page=64, lens=7),
        # one long sequence handed over to a dense kernel
        dict(name="read_1x1500_bf16", op="read", type="bf16", cache="bf16", seqs=1, kv_lo=1500, kv_hi=1500,
             kv_heads=8, dim=128, page=16, lens=8),
        # a batch of 8-bit sequences
        dict(name="read_16x8k_e4m3", op="read", type="bf16", cache="e4m3", seqs=16, kv_lo=100, kv_hi=8192,
             kv_heads=8, dim=128, page=32, lens=9),
        # the norm of a decode step, one scale a row for the projection that follows: latency
        dict(name="norm8_64x4096_row", op="norm8", type="bf16", rows=64, width=4096, group=0),
        # the same for a prefill step, a scale for every 128 columns
        dict(name="norm8_16384x4096_128", op="norm8", type="bf16", rows=16384, width=4096, group=128),
        # a training step through the norm, a width that is no power of two
        dict(name="norm_train_8192x5000", op="norm", type="bf16", rows=8192, width=5000),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "write", "read", "norm8", "norm"])
    lens = rng.randrange(1 << 20)
    if op in ("norm8", "norm"):
        width = _spread(rng, 64, 16384)
        width -= width % rng.choice([1, 2, 8, 8, 8])
        c = dict(op=op, type=rng.choice(["bf16", "bf16", "fp16", "fp32"]), rows=_spread(rng, 1, (1 << 25) // width), width=max(1, width))
        if op == "norm8":
            c["group"] = rng.choice([0, 32, 64, 128])
        return c
    cache = rng.choice(["same", "e4m3"])
    kind = rng.choice(["bf16", "fp16"])
    c = dict(op=op, type=kind, cache=kind if cache == "same" else cache, kv_heads=rng.choice([1, 2, 4, 8]), dim=rng.choice([64, 128]),
             page=rng.choice([16, 32, 64, 128]), lens=lens)
    if op == "attend":
        c["heads"] = c["kv_heads"] * rng.choice([1, 2, 3, 4, 6, 7, 8])
        way = rng.choice(["token", "draft", "chunk", "mixed"])
        if way in ("token", "draft"):
            c.update(seqs=_spread(rng, 1, 64), q=1 if way == "token" else rng.randint(2, 16), long_q=0)
            hi = _spread(rng, 64, 16384)
        elif way == "chunk":
            c.update(seqs=rng.randint(1, 2), q=_spread(rng, 17, 1400), long_q=0)
            hi = c["q"] + _spread(rng, 1, 2600)
        else:
            c.update(seqs=rng.randint(2, 16), q=rng.randint(1, 4), long_q=_spread(rng, 32, 700))
            hi = c["long_q"] + _spread(rng, 1, 3000)
        c.update(kv_lo=max(c["q"], c["long_q"]), kv_hi=max(hi, c["q"], c["long_q"]))
        return c
    c.update(seqs=_spread(rng, 1, 64), kv_hi=_spread(rng, 64, 4096))
    c["kv_lo"] = rng.randint(1, c["kv_hi"])
    if op == "write":
        c.update(q=rng.choice([1, 1, 3, c["kv_lo"]]), long_q=0)
        c["q"] = min(c["q"], c["kv_lo"])
    return c


def _lengths(case):
    """(new tokens, positions) of every sequence; a case has the same ones whatever the seed."""
    r = random.Random(case["lens"])
    kv = [r.randint(case["kv_lo"], case["kv_hi"]) for _ in range(case["seqs"])]
    q = [case.get("q", 0)] * case["seqs"]
    if case.get("long_q"):
        q[r.randrange(case["seqs"])] = case["long_q"]
    elif case.get("q", 0) > 16:   # chunks of a prompt end where the prompt does
        q = [max(1, n - r.randrange(n // 4)) for n in q]
    return q, kv


# ---------------------------------------------------------------- work

def work(case):
    es = SIZES[case["type"]]
    if case["op"] == "norm8":
        n = case["rows"] * case["width"]
        groups = case["rows"] * (-(-case["width"] // case["group"]) if case["group"] else 1)
        return {"bytes": n * (3 * es + 1) + 4 * groups + case["width"] * es, "flops": 8 * n}
    if case["op"] == "norm":
        n = case["rows"] * case["width"]   # forward: x, r -> h, y; backward: gy, gh, h -> gx
        return {"bytes": n * 8 * es + 3 * case["width"] * es, "flops": 20 * n}
    q, kv = _lengths(case)
    cs = SIZES[case["cache"]] * case["dim"] + (1 if case["cache"] == "e4m3" else 0)
    row = 2 * case["kv_heads"]   # a position's rows: keys and values of every kv head
    if case["op"] == "write":
        return {"bytes": sum(q) * row * (case["dim"] * es + cs), "flops": 3 * sum(q) * row * case["dim"]}
    if case["op"] == "read":
        return {"bytes": sum(kv) * row * (case["dim"] * es + cs), "flops": sum(kv) * row * case["dim"]}
    pairs = sum(n * k - n * (n - 1) // 2 for n, k in zip(q, kv))
    return {"bytes": 2 * sum(q) * case["heads"] * case["dim"] * es + sum(kv) * row * cs, "flops": 4 * case["heads"] * case["dim"] * pairs}


# ---------------------------------------------------------------- inputs

def _quantise(x):
    """Rows of x in 8 bits: (e4m3 values, exponent bytes)."""
    x = x.float()
    m, e = torch.frexp(x.abs().amax(-1))           # amax = m * 2^e, m in [0.5, 1): 448 = 0.875 * 2^9
    e = torch.where(m > 0.875, e - 8, e - 9).clamp(E_LO, E_HI)
    e = torch.where(m == 0, torch.zeros_like(e), e)
    v = torch.ldexp(x, -e.unsqueeze(-1)).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return v, (e + 127).to(torch.uint8)


def _values(cache, exps):
    """What a cache stands for, in fp32."""
    v = cache.float()
    return v if exps is None else torch.ldexp(v, exps.to(torch.int32).unsqueeze(-1) - 127)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = TYPES[case["type"]]

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device=DEV).mul_(scale)

    if case["op"] in ("norm8", "norm"):
        shape = (case["rows"], case["width"])
        s = {"case": case, "x": normal(*shape).to(dt), "r": normal(*shape, scale=3.0).to(dt),
             "w": (1 + normal(case["width"], scale=0.1)).to(dt), "eps": 1e-6}
        if case["op"] == "norm":
            s["gy"], s["gh"] = normal(*shape).to(dt), normal(*shape).to(dt)
        return s
    q_lens, kv_lens = _lengths(case)
    page, H, D, B = case["page"], case["kv_heads"], case["dim"], case["seqs"]
    need = [-(-n // page) for n in kv_lens]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    table = torch.full((B, max(need)), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    s = {"case": case, "table": table, "kv_lens": torch.tensor(kv_lens, dtype=torch.int32, device=DEV), "total": sum(kv_lens),
         "cu_q": torch.tensor([sum(q_lens[:i]) for i in range(B + 1)], dtype=torch.int32, device=DEV),
         "cu_kv": torch.tensor([sum(kv_lens[:i]) for i in range(B + 1)], dtype=torch.int32, device=DEV),
         "max_q": max(q_lens), "scale": D ** -0.5}
    # keys with a few large channels, as projections have them; values around one
    wide = torch.exp(normal(D, scale=0.5))
    for name in ("k", "v"):
        if case["op"] == "write":
            c = torch.zeros(pages, H, page, D, device=DEV, dtype=torch.uint8 if case["cache"] == "e4m3" else dt)
            s[name] = (normal(sum(q_lens), H, D) * wide).to(dt)
        else:
            c = torch.empty(pages, H, page, D, dtype=dt, device=DEV)
            step = max(1, (1 << 26) // (H * page * D))
            for i in range(0, pages, step):
                n = min(step, pages - i)
                c[i:i + n] = (normal(n, H, page, D) * (wide if name == "k" else 1.0)).to(dt)
        e = None
        if case["cache"] == "e4m3":
            if case["op"] == "write":
                c, e = c.view(torch.float8_e4m3fn), torch.zeros(pages, H, page, dtype=torch.uint8, device=DEV)
            else:
                step = max(1, (1 << 26) // (H * page * D))
                parts = [_quantise(c[i:i + step]) for i in range(0, pages, step)]
                c = torch.cat([p[0].view(torch.uint8) for p in parts]).view(torch.float8_e4m3fn)
                e = torch.cat([p[1] for p in parts])
        s[name + "_cache"], s[name + "_exp"] = c, e
    if case["op"] == "attend":
        s["q"] = normal(sum(q_lens), case["heads"], D).to(dt)
    return s


# ---------------------------------------------------------------- the plain forms

def _rows_of(cu, count):
    """(sequence, place in it) of each of `count` ragged rows."""
    t = torch.arange(count, device=cu.device)
    b = torch.searchsorted(cu.long(), t, right=True) - 1
    return b, t - cu.long()[b]


def _pages(cache, table):
    """Pages by number, whatever their type; absent ones read as some page."""
    i = table.long().clamp_min(0)
    return cache.view(torch.uint8)[i].view(cache.dtype) if cache.dtype == torch.float8_e4m3fn else cache[i]


def _dense(cache, exps, table):
    """[B, kv heads, positions, D] in fp32."""
    v = _values(_pages(cache, table), None if exps is None else exps[table.long().clamp_min(0)])
    v = v.transpose(1, 2)
    return v.reshape(v.shape[0], v.shape[1], -1, v.shape[-1])


def _attend(s):
    q, cu, kv = s["q"], s["cu_q"].long(), s["kv_lens"].long()
    T, H, D = q.shape
    k, v = _dense(s["k_cache"], s["k_exp"], s["table"]), _dense(s["v_cache"], s["v_exp"], s["table"])
    B, Hk, L = k.shape[:3]
    n = s["max_q"]
    i = torch.arange(n, device=q.device)
    rows = (cu[:-1, None] + i).clamp_max(T - 1)
    qp = q[rows].float().mul(s["scale"]).view(B, n, Hk, H // Hk, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, -1, D)
    last = (kv - (cu[1:] - cu[:-1]))[:, None] + i            # the last position that row i attends
    hidden = torch.arange(L, device=q.device) > torch.minimum(last, kv[:, None] - 1)[..., None]
    x = torch.matmul(qp, k.transpose(-1, -2)).view(B, Hk, H // Hk, n, L).masked_fill_(hidden[:, None, None], float("-inf"))
    x = x.sub_(x.amax(-1, keepdim=True)).exp_()
    x = x.div_(x.sum(-1, keepdim=True)).view(B, Hk, -1, L)
    o = torch.matmul(x, v).view(B, H, n, D)
    b, at = _rows_of(cu, T)
    return o[b, :, at].to(q.dtype)


def _write(s):
    b, at = _rows_of(s["cu_q"], s["k"].shape[0])
    cu, page = s["cu_q"].long(), s["k_cache"].shape[2]
    pos = s["kv_lens"].long()[b] - (cu[1:] - cu[:-1])[b] + at
    where, off = s["table"].long()[b, pos // page], pos % page
    out = []
    for x, cache, exps in ((s["k"], s["k_cache"], s["k_exp"]), (s["v"], s["v_cache"], s["v_exp"])):
        if exps is None:
            cache[where, :, off] = x
            out += [cache]
        else:
            v, e = _quantise(x)
            cache.view(torch.uint8)[where, :, off] = v.view(torch.uint8)
            exps[where, :, off] = e
            out += [cache, exps]
    return out


def _read(s):
    b, at = _rows_of(s["cu_kv"], s["total"])
    page = s["k_cache"].shape[2]
    where, off = s["table"].long()[b, at // page], at % page
    out = []
    for cache, exps in ((s["k_cache"], s["k_exp"]), (s["v_cache"], s["v_exp"])):
        if exps is None:
            out.append(cache[where, :, off])
        else:
            rows = cache.view(torch.uint8)[where, :, off].view(torch.float8_e4m3fn)
            out.append(_values(rows, exps[where, :, off]).to(TYPES[s["case"]["type"]]))
    return out


def _norm(s):
    h = (s["x"].float() + s["r"].float()).to(s["x"].dtype)
    hf = h.float()
    rstd = torch.rsqrt(hf.double().square().mean(-1, keepdim=True) + s["eps"]).float()
    return h, hf, rstd, hf * rstd * s["w"].float()


def _norm8(s, group):
    h, _, _, y = _norm(s)
    rows, width = y.shape
    g = group or width
    n = -(-width // g)
    y = torch.nn.functional.pad(y, (0, n * g - width)).view(rows, n, g)
    scale = (y.abs().amax(-1) / 448.0).clamp_min(2.0 ** -126)
    q = (y / scale.unsqueeze(-1)).clamp(-448.0, 448.0).view(rows, -1)[:, :width].to(torch.float8_e4m3fn)
    return [h, q, scale]


def _norm_train(s):
    h, hf, rstd, y = _norm(s)
    gy, w = s["gy"].float(), s["w"].float()
    gw_ = gy * w
    n = hf * rstd
    gx = rstd * (gw_ - n * (gw_ * n).mean(-1, keepdim=True)) + s["gh"].float()
    gw = (gy * n).double().sum(0)
    return [h, y.to(h.dtype), gx.to(h.dtype), gw.to(h.dtype)]


def run(state):
    s, op = state, state["case"]["op"]
    if own:
        abi = _abi()
        if op == "attend":
            return abi.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["kv_lens"], s["cu_q"], s["max_q"],
                                       scale=s["scale"], k_exp=s["k_exp"], v_exp=s["v_exp"])
        if op == "write":
            abi.paged_kv_write(s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["kv_lens"], s["cu_q"],
                               k_exp=s["k_exp"], v_exp=s["v_exp"])
            return [x for n in ("k", "v") for x in (s[n + "_cache"], s[n + "_exp"]) if x is not None]
        if op == "read":
            return list(abi.paged_kv_read(s["k_cache"], s["v_cache"], s["table"], s["cu_kv"], s["total"],
                                          dtype=TYPES[s["case"]["type"]], k_exp=s["k_exp"], v_exp=s["v_exp"]))
        if op == "norm8":
            q, scale, h = abi.add_rmsnorm_quant(s["x"], s["r"], s["w"], s["eps"], group=s["case"]["group"])
            return [h, q, scale]
        y, h, rstd = abi.add_rmsnorm_fwd(s["x"], s["r"], s["w"], s["eps"], return_rstd=True)
        gx, gw = abi.add_rmsnorm_bwd(s["gy"], s["gh"], h, s["w"], rstd)
        return [h, y, gx, gw]
    if op == "attend":
        return _attend(s)
    if op == "write":
        return _write(s)
    if op == "read":
        return _read(s)
    if op == "norm8":
        return _norm8(s, s["case"]["group"])
    return _norm_train(s)


# ---------------------------------------------------------------- the definition, in 64 bits

def _exact_rows(cache, exps, pages, count):
    """The first `count` positions on these pages, [kv heads, count, D]."""
    i = pages.long()
    v = cache.view(torch.uint8)[i].view(cache.dtype) if exps is not None else cache[i]
    v = v.to(torch.float32).double()
    if exps is not None:
        v = v * torch.pow(2.0, exps[i].double() - 127).unsqueeze(-1)
    return torch.cat(list(v), dim=1)[:, :count]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("norm8", "norm"):
        h = (s["x"].double() + s["r"].double()).to(s["x"].dtype)   # the sum is kept in the type
        hd, w = h.double(), s["w"].double()
        r = 1.0 / torch.sqrt((hd * hd).sum(1, keepdim=True) / case["width"] + s["eps"])
        y = hd * r * w
        if case["op"] == "norm8":
            g = case["group"] or case["width"]
            top = torch.stack([y[:, i:i + g].abs().amax(1) for i in range(0, case["width"], g)], 1) / 448.0
            top = top.clamp_min(2.0 ** -126)
            return [s["x"].double() + s["r"].double(), y / torch.repeat_interleave(top, g, 1)[:, :case["width"]], top]
        gy, gh = s["gy"].double(), s["gh"].double()
        a = gy * w
        gx = r * a - hd * r ** 3 * (a * hd).sum(1, keepdim=True) / case["width"] + gh
        return [s["x"].double() + s["r"].double(), y, gx, (gy * hd * r).sum(0)]
    q_lens, kv_lens = _lengths(case)
    page = case["page"]
    if case["op"] == "write":
        out = []
        for name in ("k", "v"):
            c, e = s[name + "_cache"].float().double(), s[name + "_exp"]
            e = None if e is None else e.long()
            t = 0
            for b in range(case["seqs"]):
                pos = torch.arange(kv_lens[b] - q_lens[b], kv_lens[b], device=DEV)
                x = s[name][t:t + q_lens[b]].double()
                t += q_lens[b]
                where = s["table"][b].long()[pos // page]
                if e is not None:
                    top = x.abs().amax(-1)
                    x2 = torch.ceil(torch.log2(top.clamp_min(1e-300) / 448.0)).clamp(E_LO, E_HI)
                    x2 = torch.where(top == 0, torch.zeros_like(x2), x2)
                    e[where, :, pos % page] = x2.long() + 127
                    x = x / torch.pow(2.0, x2).unsqueeze(-1)
                c[where, :, pos % page] = x
            out.append(c)
            if e is not None:
                out.append(None)
        return out
    if case["op"] == "read":
        out = []
        for name in ("k", "v"):
            rows = [_exact_rows(s[name + "_cache"], s[name + "_exp"], s["table"][b, :-(-n // page)], n) for b, n in enumerate(kv_lens)]
            out.append(torch.cat(rows, 1).transpose(0, 1))
        return out
    group, out, t = case["heads"] // case["kv_heads"], [], 0
    for b, (n, L) in enumerate(zip(q_lens, kv_lens)):
        k, v = (_exact_rows(s[x + "_cache"], s[x + "_exp"], s["table"][b, :-(-L // page)], L) for x in ("k", "v"))
        q = s["q"][t:t + n].double()
        t += n
        o = torch.empty(n, case["heads"], case["dim"], dtype=torch.float64, device=DEV)
        later = torch.arange(L, device=DEV)[None] > torch.arange(L - n, L, device=DEV)[:, None]
        for h in range(case["heads"]):
            x = q[:, h] @ k[h // group].T * s["scale"]
            x[later] = float("-inf")
            o[:, h] = torch.softmax(x, -1) @ v[h // group]
        out.append(o)
    return torch.cat(out)
