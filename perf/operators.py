"""What is measured of the paged-cache serving operators: causal attention over
packed prompts, attention of new tokens over a paged cache, the page planner
and the norm + RoPE + cache-write prologue.

With `own` false, `run` computes the operators in plain torch (fp32
arithmetic, rounded once at the end); with `own` true it makes the calls a
user makes. Sizes are those of grouped-head text models (32 query and 8 key
heads of 128; 14 and 2 of 64; 28 and 4 of 128).
"""
import math
import os
import random
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_DT = {"bf16": torch.bfloat16, "f16": torch.float16}


def _lib():
    """The package, as a user's program imports it."""
    path = os.path.join(_ROOT, "llm-runner_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import llmr_attn
    return llmr_attn


# ------------------------------------------------------------------- cases

def listed():
    return [
        # One image prompt through a text encoder: the call's latency counts.
        dict(name="causal_prompt77", op="causal", n=1, lo=77, hi=77, mix=1, heads=32, kv_heads=8,
             dim=128, dtype="bf16", lse=False),
        # A batch of prompts of very different lengths, odd group of 7, small heads.
        dict(name="causal_ragged", op="causal", n=24, lo=1, hi=1500, mix=2, heads=14, kv_heads=2,
             dim=64, dtype="f16", lse=True),
        # One long document: the largest prompt.
        dict(name="causal_8k", op="causal", n=1, lo=8192, hi=8192, mix=3, heads=32, kv_heads=8,
             dim=128, dtype="bf16", lse=False),
        # A single user's next token over a short context: latency again.
        dict(name="decode_one", op="paged", n=1, qlo=1, qhi=1, lo=1500, hi=1500, mix=4, heads=32,
             kv_heads=8, dim=128, page=16, dtype="bf16", pad=0, lse=False),
        # A serving step: 64 requests, one token each, contexts of all lengths;
        # the batch is padded to the captured graph's size.
        dict(name="decode_batch64", op="paged", n=64, qlo=1, qhi=1, lo=130, hi=9000, mix=5,
             heads=32, kv_heads=8, dim=128, page=16, dtype="bf16", pad=8, lse=False),
        # Five drafted tokens per request to verify, group of 7.
        dict(name="draft5", op="paged", n=24, qlo=5, qhi=5, lo=300, hi=6000, mix=6, heads=28,
             kv_heads=4, dim=128, page=32, dtype="f16", pad=0, lse=True),
        # Chunked prefill: chunks of prompts behind long cached prefixes.
        dict(name="chunk_prefill", op="paged", n=6, qlo=300, qhi=700, lo=2000, hi=12000, mix=7,
             heads=32, kv_heads=8, dim=128, page=64, dtype="bf16", pad=0, lse=False),
        # One last chunk over a long prefix, small heads, few heads: the long
        # axis has to be split to fill the card.
        dict(name="chunk_long_prefix", op="paged", n=1, qlo=129, qhi=129, lo=50001, hi=50001,
             mix=8, heads=14, kv_heads=2, dim=64, page=16, dtype="f16", pad=0, lse=False),
        # Planning a serving step, and planning a prefill step.
        dict(name="plan_decode", op="plan", n=256, new_lo=1, new_hi=1, ctx_hi=8000, mix=9, page=16),
        dict(name="plan_prefill", op="plan", n=48, new_lo=1, new_hi=4000, ctx_hi=3000, mix=10,
             page=64),
        # The step before a decode's attention, and before a prefill's.
        dict(name="prologue_decode", op="prologue", tokens=64, heads=32, kv_heads=8, dim=128,
             page=16, dtype="bf16", norm=True, half=True),
        dict(name="prologue_prefill", op="prologue", tokens=8191, heads=32, kv_heads=8, dim=128,
             page=64, dtype="bf16", norm=True, half=False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


_HEADS = ((32, 8, 128), (14, 2, 64), (28, 4, 128), (16, 16, 64), (8, 1, 128), (12, 4, 128),
          (40, 8, 64), (16, 8, 128))


def draw(rng):
    op = rng.choice(("causal", "causal", "paged", "paged", "paged", "plan", "prologue"))
    heads, kv_heads, dim = rng.choice(_HEADS)
    dtype = rng.choice(("bf16", "f16"))
    mix = rng.randrange(1 << 30)
    page = rng.choice((16, 32, 64, 128))
    base = dict(op=op, mix=mix)
    if op == "causal":
        n = _log_int(rng, 1, 32)
        hi = _log_int(rng, 2, 7000 // n + 2)
        return dict(base, n=n, lo=rng.randrange(1, hi + 1) if rng.random() < 0.5 else 1, hi=hi,
                    heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype,
                    lse=rng.random() < 0.5)
    if op == "paged":
        kind = rng.choice(("decode", "few", "chunk"))
        n = _log_int(rng, 1, {"decode": 64, "few": 32, "chunk": 6}[kind])
        qhi = {"decode": 1, "few": rng.randrange(2, 17), "chunk": _log_int(rng, 17, 700)}[kind]
        hi = _log_int(rng, 200, min(50000, 250000 // n if kind == "decode" else 40000 // n))
        return dict(base, n=n, qlo=1 if kind == "decode" else rng.randrange(1, qhi + 1), qhi=qhi,
                    lo=rng.randrange(1, hi + 1), hi=hi, heads=heads, kv_heads=kv_heads, dim=dim,
                    page=page, dtype=dtype, pad=rng.choice((0, 0, 3)), lse=rng.random() < 0.5)
    if op == "plan":
        n = _log_int(rng, 1, 512)
        return dict(base, n=n, new_lo=rng.randrange(0, 2), new_hi=_log_int(rng, 1, 60000 // n + 1),
                    ctx_hi=_log_int(rng, 1, 9000), page=page)
    return dict(op=op, tokens=_log_int(rng, 1, 8191), heads=heads, kv_heads=kv_heads, dim=dim,
                page=page, dtype=dtype, norm=rng.random() < 0.7, half=rng.random() < 0.5)


def _spread(rng, n, lo, hi):
    """n lengths, spread over the logarithm of [lo, hi]."""
    return [_log_int(rng, lo, hi) if hi > 0 else 0 for _ in range(n)]


def _lens(case):
    """(new tokens, total keys) of each request: part of the case, not of the seed."""
    rng = random.Random(case["mix"])
    if case["op"] == "causal":
        lens = _spread(rng, case["n"], case["lo"], case["hi"])
        return lens, lens
    if case["op"] == "paged":
        q = [rng.randint(case["qlo"], case["qhi"]) for _ in range(case["n"])]
        kv = _spread(rng, case["n"], case["lo"], case["hi"])
        return q, [max(a, b) for a, b in zip(q, kv)]
    new = [rng.randint(case["new_lo"], case["new_hi"]) for _ in range(case["n"])]
    ctx = [rng.randint(0, case["ctx_hi"]) for _ in range(case["n"])]
    return new, [a + b for a, b in zip(new, ctx)]


def work(case):
    """Bytes and operations one pass cannot do without."""
    op = case["op"]
    if op in ("causal", "paged"):
        q, kv = _lens(case)
        h, hk, d = case["heads"], case["kv_heads"], case["dim"]
        pairs = sum(b * (b + 1) // 2 - (b - a) * (b - a + 1) // 2 for a, b in zip(q, kv))
        moved = 2 * 2 * sum(q) * h * d + 2 * 2 * sum(kv) * hk * d + (4 * sum(q) * h if case["lse"] else 0)
        if op == "paged":
            moved += 4 * sum(-(-b // case["page"]) for b in kv)
        return {"bytes": moved, "flops": 4 * pairs * h * d}
    if op == "plan":
        new, tot = _lens(case)
        p = case["page"]
        fresh = sum(-(-t // p) - -(-(t - n) // p) for n, t in zip(new, tot))
        # lengths in, offsets and totals out; a slot and a position per token;
        # each new page read from the free list and written to the table
        return {"bytes": 4 * (4 * len(new) + 3 + 2 * sum(new) + 2 * fresh), "flops": 0}
    rows = case["tokens"] * (case["heads"] + 2 * case["kv_heads"]) * case["dim"]
    return {"bytes": 2 * 2 * rows + 8 * case["tokens"] + 4 * case["tokens"] * case["dim"],
            "flops": 10 * rows}


# ------------------------------------------------------------------ inputs

def _randn(g, *shape, dtype):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _cumulative(lens):
    out = [0]
    for x in lens:
        out.append(out[-1] + x)
    return out


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    s = {"case": case}
    if own:
        L = _lib()
        s["L"], s["ctx"] = L, L.Context(torch.cuda.current_device())
    if op in ("causal", "paged"):
        dt, h, hk, d = _DT[case["dtype"]], case["heads"], case["kv_heads"], case["dim"]
        q_lens, kv_lens = _lens(case)
        tokens = sum(q_lens) + case.get("pad", 0)
        s.update(scale=d ** -0.5, cu=_ints(_cumulative(q_lens)), q=_randn(g, tokens, h, d, dtype=dt),
                 o=torch.zeros((tokens, h, d), dtype=dt, device="cuda"),
                 lse=torch.zeros((h, tokens), device="cuda") if case["lse"] else None)
        if op == "causal":
            s.update(k=_randn(g, tokens, hk, d, dtype=dt), v=_randn(g, tokens, hk, d, dtype=dt))
            return s
        page = case["page"]
        pages = [-(-x // page) for x in kv_lens]
        num_pages = sum(pages) + 5
        table = torch.zeros((len(pages), max(pages)), dtype=torch.int32)
        order = torch.randperm(num_pages, generator=torch.Generator().manual_seed(seed)).int()
        at = 0
        for i, x in enumerate(pages):
            table[i, :x] = order[at:at + x]
            at += x
        s.update(kv_lens=_ints(kv_lens), table=table.cuda(), max_q=max(q_lens), max_kv=max(kv_lens),
                 k_cache=_randn(g, num_pages, page, hk, d, dtype=dt),
                 v_cache=_randn(g, num_pages, page, hk, d, dtype=dt))
        if own:
            s["ctx"].reserve(s["L"].attention_paged_workspace_bytes(
                n_seqs=len(q_lens), total_tokens=tokens, max_q_len=s["max_q"], n_heads=h,
                n_kv_heads=hk, head_dim=d))
        return s
    if op == "plan":
        new, tot = _lens(case)
        page = case["page"]
        ctx_lens = [t - n for n, t in zip(new, tot)]
        held = [-(-c // page) for c in ctx_lens]
        need = [-(-t // page) - a for t, a in zip(tot, held)]
        cols = max(1, max(a + b for a, b in zip(held, need)))
        order = torch.randperm(sum(held) + sum(need) + 37,
                               generator=torch.Generator().manual_seed(seed)).int()
        table = torch.full((len(new), cols), -1, dtype=torch.int32)
        at = 0
        for i, a in enumerate(held):
            table[i, :a] = order[at:at + a]
            at += a
        room = sum(new) + 16   # the arrays of a captured step are longer than most steps need
        s.update(ctx_lens=_ints(ctx_lens), new_lens=_ints(new), free=order[at:].cuda(),
                 n_free=_ints([len(order) - at]), table=table.cuda(), page=page, room=room)
        if own:
            new_int = lambda k: torch.zeros(k, dtype=torch.int32, device="cuda")
            s.update(cu=new_int(len(new) + 1), kv_lens=new_int(len(new)), positions=new_int(room),
                     slots=new_int(room), n_free_out=new_int(1))
        return s
    dt, h, hk, d, page = (_DT[case["dtype"]], case["heads"], case["kv_heads"], case["dim"],
                          case["page"])
    t = case["tokens"]
    num_pages = -(-t // page) + 9
    rows = 9000
    host = torch.Generator().manual_seed(seed)
    angle = (torch.arange(rows, dtype=torch.float64)[:, None]
             * 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)[None])
    s.update(qkv=_randn(g, t, (h + 2 * hk) * d, dtype=dt), cos=angle.cos().float().cuda(),
             sin=angle.sin().float().cuda(),
             q_gain=torch.rand(d, generator=g, device="cuda") * 0.4 + 0.8,
             k_gain=torch.rand(d, generator=g, device="cuda") * 0.4 + 0.8,
             positions=torch.randint(0, rows, (t,), generator=host, dtype=torch.int32).cuda(),
             slots=torch.randperm(num_pages * page, generator=host)[:t].int().cuda(),
             q_out=torch.zeros((t, h, d), dtype=dt, device="cuda"),
             k_cache=torch.zeros((num_pages, page, hk, d), dtype=dt, device="cuda"),
             v_cache=torch.zeros((num_pages, page, hk, d), dtype=dt, device="cuda"), eps=1e-6)
    return s


# --------------------------------------------------------------- one pass

def run(s):
    op = s["case"]["op"]
    return {"causal": _causal, "paged": _paged, "plan": _plan, "prologue": _prologue}[op](s)


def _outs(o, lse):
    return {"o": o} if lse is None else {"o": o, "lse": lse}


def _owner(cu, tokens):
    """Which sequence each packed row belongs to (n for rows behind the last), and its index there."""
    row = torch.arange(tokens, device=cu.device)
    seq = torch.searchsorted(cu[1:].long(), row, right=True)
    return seq, row - cu.long()[seq]


def _masked_softmax(x, keep):
    """exp(x - max) over the kept entries of the last axis, its sum, and log-sum-exp."""
    x = torch.where(keep, x, -math.inf)
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    e = (x - top).exp()
    total = e.sum(-1, keepdim=True)
    return e, total, (total.log() + top)[..., 0]


def _causal(s):
    if own:
        s["L"].attention_causal(s["ctx"], s["q"], s["k"], s["v"], s["o"], s["cu"], scale=s["scale"],
                                lse=s["lse"])
        return _outs(s["o"], s["lse"])
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    t, h, d = q.shape
    hk = k.shape[1]
    seq, idx = _owner(s["cu"], t)
    keep = (seq[:, None] == seq[None]) & (idx[None] <= idx[:, None])
    x = torch.matmul(q.view(t, hk, h // hk, d).permute(1, 2, 0, 3),
                     k.permute(1, 2, 0)[:, None]) * s["scale"]          # [hk, g, t, t]
    e, total, lse = _masked_softmax(x, keep)
    o = torch.matmul(e, v.permute(1, 0, 2)[:, None]) / total
    o = o.permute(2, 0, 1, 3).reshape(t, h, d)
    return _outs(o.to(s["q"].dtype), None if s["lse"] is None else lse.reshape(h, t))


def _paged(s):
    if own:
        s["L"].attention_paged(s["ctx"], s["q"], s["k_cache"], s["v_cache"], s["o"], s["cu"],
                               s["kv_lens"], s["table"], scale=s["scale"], max_q_len=s["max_q"],
                               lse=s["lse"])
        return _outs(s["o"], s["lse"])
    t, h, d = s["q"].shape
    n, cols = s["table"].shape
    page, hk = s["k_cache"].shape[1:3]
    pages = s["table"].long()
    k = s["k_cache"][pages].float().view(n, cols * page, hk, d)[:, :s["max_kv"]]
    v = s["v_cache"][pages].float().view(n, cols * page, hk, d)[:, :s["max_kv"]]
    cu = s["cu"].long()
    q_len = cu[1:] - cu[:-1]
    idx = torch.arange(s["max_q"], device="cuda")
    row = (cu[:-1, None] + idx).clamp(max=t - 1)                         # [n, max_q]
    q = s["q"].float()[row].view(n, s["max_q"], hk, h // hk, d)
    pos = (s["kv_lens"].long() - q_len)[:, None] + idx
    key = torch.arange(s["max_kv"], device="cuda")
    keep = (key <= pos[..., None])[:, None, None]                        # [n, 1, 1, max_q, max_kv]
    x = torch.matmul(q.permute(0, 2, 3, 1, 4), k.permute(0, 2, 3, 1)[:, :, None]) * s["scale"]
    e, total, lse = _masked_softmax(x, keep)
    o = torch.matmul(e, v.permute(0, 2, 1, 3)[:, :, None]) / total       # [n, hk, g, max_q, d]
    seq, at = _owner(s["cu"], t)
    inside = seq < n
    seq, at = seq.clamp(max=n - 1), at.clamp(0, s["max_q"] - 1)
    o = o.permute(0, 3, 1, 2, 4).reshape(n, s["max_q"], h, d)[seq, at].to(s["q"].dtype)
    o = torch.where(inside[:, None, None], o, s["o"])
    if s["lse"] is None:
        return {"o": o}
    lse = lse.permute(1, 2, 0, 3).reshape(h, n, s["max_q"])[:, seq, at]
    return {"o": o, "lse": torch.where(inside, lse, s["lse"])}


def _plan(s):
    if own:
        s["L"].paged_plan(s["ctx"], s["ctx_lens"], s["new_lens"], s["free"], s["n_free"],
                          s["table"], s["cu"], s["kv_lens"], s["positions"], s["slots"],
                          s["n_free_out"], page_size=s["page"])
        return {"table": s["table"], "cu": s["cu"], "kv_lens": s["kv_lens"],
                "positions": s["positions"], "slots": s["slots"], "n_free": s["n_free_out"]}
    page, room = s["page"], s["room"]
    ctx, new = s["ctx_lens"].long(), s["new_lens"].long()
    total = ctx + new
    held, last = (ctx + page - 1) // page, (total + page - 1) // page
    taken = (last - held).cumsum(0)
    cu = torch.nn.functional.pad(new.cumsum(0), (1, 0))
    col = torch.arange(s["table"].shape[1], device="cuda")
    fresh = (col >= held[:, None]) & (col < last[:, None])
    rank = (taken - (last - held))[:, None] + col - held[:, None]
    source = (s["n_free"].long() - 1 - rank).clamp(0, s["free"].numel() - 1)
    table = torch.where(fresh, s["free"][source], s["table"])
    seq, idx = _owner(cu, room)
    live = seq < new.numel()
    seq = seq.clamp(max=new.numel() - 1)
    pos = torch.where(live, ctx[seq] + idx, 0)
    slot = table[seq, pos // page].long() * page + pos % page
    return {"table": table, "cu": cu.int(), "kv_lens": total.int(), "positions": pos.int(),
            "slots": torch.where(live, slot, -1).int(), "n_free": (s["n_free"] - taken[-1]).int()}


def _rotate(x, cos, sin, half):
    if half:
        a, b = x.chunk(2, -1)
        return torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)


def _prologue(s):
    c = s["case"]
    h, hk, d = c["heads"], c["kv_heads"], c["dim"]
    t = c["tokens"]
    q, k, v = (x.view(t, -1, d) for x in s["qkv"].split((h * d, hk * d, hk * d), 1))
    if own:
        s["L"].paged_prologue(s["ctx"], q, k, v, s["q_out"], s["k_cache"], s["v_cache"],
                              s["positions"], s["slots"], eps=s["eps"],
                              q_gain=s["q_gain"] if c["norm"] else None,
                              k_gain=s["k_gain"] if c["norm"] else None, cos=s["cos"],
                              sin=s["sin"], half=c["half"])
        return {"q": s["q_out"], "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    at = s["positions"].long()
    cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]
    q, k = q.float(), k.float()
    if c["norm"]:
        q = q * torch.rsqrt((q * q).mean(-1, keepdim=True) + s["eps"]) * s["q_gain"]
        k = k * torch.rsqrt((k * k).mean(-1, keepdim=True) + s["eps"]) * s["k_gain"]
    slots = s["slots"].long()
    s["k_cache"].view(-1, hk, d)[slots] = _rotate(k, cos, sin, c["half"]).to(v.dtype)
    s["v_cache"].view(-1, hk, d)[slots] = v
    return {"q": _rotate(q, cos, sin, c["half"]).to(v.dtype), "k_cache": s["k_cache"],
            "v_cache": s["v_cache"]}


# ------------------------------------------------------ the definition, 64 bits

def exact(case, seed):
    """The outputs from the definitions in 64 bits, request by request and row block by row block.

    A plan's outputs are whole numbers, for which the plain form is the definition."""
    global own
    if case["op"] == "plan":
        return None
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    op = case["op"]
    d = case["dim"]
    h, hk = case["heads"], case["kv_heads"]
    group = h // hk
    if op == "prologue":
        out = {"k_cache": s["k_cache"].double().cpu(), "v_cache": s["v_cache"].double().cpu()}
        x = s["qkv"].double().cpu().view(case["tokens"], h + 2 * hk, d)
        angle_cos, angle_sin = s["cos"].double().cpu(), s["sin"].double().cpu()
        pos, slots = s["positions"].long().cpu(), s["slots"].long().cpu()
        c, sn = angle_cos[pos].unsqueeze(1), angle_sin[pos].unsqueeze(1)
        turned = []
        for part, gain in ((x[:, :h], s["q_gain"]), (x[:, h:h + hk], s["k_gain"])):
            if case["norm"]:
                part = part / (part.pow(2).sum(-1, keepdim=True) / d + s["eps"]).sqrt()
                part = part * gain.double().cpu()
            pairs = (part.reshape(*part.shape[:-1], 2, d // 2).transpose(-1, -2) if case["half"]
                     else part.reshape(*part.shape[:-1], d // 2, 2))
            z = torch.view_as_complex(pairs.contiguous()) * torch.complex(c, sn)
            flat = torch.view_as_real(z)
            turned.append((flat.transpose(-1, -2) if case["half"] else flat).reshape(part.shape))
        out["q"] = turned[0]
        out["k_cache"].view(-1, hk, d)[slots] = turned[1]
        out["v_cache"].view(-1, hk, d)[slots] = x[:, h + hk:]
        return {name: out[name] for name in ("q", "k_cache", "v_cache")}
    q_lens, kv_lens = _lens(case)
    tokens = s["q"].shape[0]
    o = torch.zeros((tokens, h, d), dtype=torch.float64, device="cuda")
    lse = torch.zeros((h, tokens), dtype=torch.float64, device="cuda")
    start = 0
    for r, (nq, nk) in enumerate(zip(q_lens, kv_lens)):
        if op == "causal":
            keys, values = s["k"][start:start + nk], s["v"][start:start + nk]
        else:
            where = s["table"][r, :-(-nk // case["page"])].long()
            keys = s["k_cache"].index_select(0, where).flatten(0, 1)[:nk]
            values = s["v_cache"].index_select(0, where).flatten(0, 1)[:nk]
        keys, values = keys.double(), values.double()
        for first in range(0, nq, 1024):
            rows = torch.arange(first, min(first + 1024, nq), device="cuda")
            hidden = torch.arange(nk, device="cuda") > (nk - nq + rows).unsqueeze(1)
            for head in range(h):
                z = s["q"][start + rows, head].double() @ keys[:, head // group].t() * s["scale"]
                z = z.masked_fill(hidden, float("-inf"))
                norm = torch.logsumexp(z, 1)
                o[start + rows, head] = torch.exp(z - norm.unsqueeze(1)) @ values[:, head // group]
                lse[head, start + rows] = norm
        start += nq
    return {"o": o, "lse": lse} if case["lse"] else {"o": o}
