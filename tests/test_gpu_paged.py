"""GPU: causal prompts, paged attention, the planner and the paged prologue
against plain 64-bit forms (paged_reference.py), at the lengths, head
layouts, strides and masks where they can go wrong, and run together as a
serving step runs them."""
import math

import pytest
import torch

import llmr_attn as L
import paged_reference as R

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def cumulative(lens):
    out = [0]
    for x in lens:
        out.append(out[-1] + x)
    return out


def randn(seed, *shape, dtype=BF16, size=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * size).to(dtype)


# ------------------------------------------------------------- causal prompts

def run_causal(ctx, lens, h, hk, d, dtype, out_dtype, *, pad=0, size=1.0, scale=None, seed=0,
               qkv=None, o=None):
    scale = scale or d ** -0.5
    t = sum(lens) + pad
    if qkv is None:
        qkv = (randn(seed, t, h, d, dtype=dtype, size=size), randn(seed + 1, t, hk, d, dtype=dtype, size=size),
               randn(seed + 2, t, hk, d, dtype=dtype))
    q, k, v = qkv
    if pad:   # rows behind the last sequence: whatever they hold must not matter
        for x in (q, k, v):
            x[t - pad:] = math.nan
    if o is None:
        o = torch.full((t, h, d), 7.0, dtype=out_dtype, device="cuda")
    lse = torch.full((h, t), 7.0, device="cuda")
    L.attention_causal(ctx, q, k, v, o, ints(cumulative(lens)), scale=scale, lse=lse)
    ctx.sync()
    at = 0
    for n in lens:
        if n:
            w, wl, weight = R.rows_attention(q[at:at + n], k[at:at + n], v[at:at + n], scale)
            R.check_attention(o[at:at + n], lse[:, at:at + n], w, wl, weight, dtype, d, n,
                              float(v[at:at + n].abs().max()),
                              R.score_size(q[at:at + n], k[at:at + n], scale), (lens, at))
        at += n
    assert (o[at:] == 7).all() and (lse[:, at:] == 7).all()
    return o


@pytest.mark.parametrize("h,hk,d", [(4, 4, 64), (8, 2, 128), (14, 2, 64), (7, 1, 128), (16, 1, 64),
                                    (6, 2, 128), (40, 8, 64)])
@pytest.mark.parametrize("lens", [[1], [77], [0, 5, 0, 300, 1, 0], [128, 129, 127], [641]])
def test_causal_lengths_and_heads(ctx, lens, h, hk, d):
    run_causal(ctx, lens, h, hk, d, BF16, BF16, pad=3, seed=len(lens))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("out_dtype", [F16, BF16, F32])
@pytest.mark.parametrize("d", [64, 128])
def test_causal_types(ctx, dtype, out_dtype, d):
    run_causal(ctx, [200, 57], 8, 4, d, dtype, out_dtype, seed=3)


def test_causal_many_sequences(ctx):
    """More sequences than a warp searches at once, most of them short or empty."""
    g = torch.Generator().manual_seed(5)
    lens = torch.randint(0, 9, (1500,), generator=g).tolist()
    lens[700] = 400
    run_causal(ctx, lens, 4, 2, 64, F16, F16, pad=2, seed=5)


def test_causal_peaked_rows(ctx):
    """Scores that jump in later key blocks move the running maximum."""
    h, hk, d, n = 4, 2, 128, 900
    q, k, v = randn(1, n, h, d), randn(2, n, hk, d), randn(3, n, hk, d)
    k[300] *= 6
    k[650] *= 12
    run_causal(ctx, [n], h, hk, d, BF16, BF16, qkv=(q, k, v))
    run_causal(ctx, [n], h, hk, d, F16, F16, qkv=(q.to(F16), k.to(F16), v.to(F16)))


def test_causal_long(ctx):
    run_causal(ctx, [5000], 4, 1, 128, BF16, BF16, seed=9)


def test_causal_strides(ctx):
    """A fused QKV buffer, head-major tensors, and an output with a gap between rows."""
    lens, h, hk, d = [130, 45], 6, 2, 64
    t = sum(lens)
    fused = randn(1, t, (h + 2 * hk) * d, dtype=F16)
    q, k, v = (x.unflatten(1, (-1, d)) for x in fused.split((h * d, hk * d, hk * d), 1))
    want = run_causal(ctx, lens, h, hk, d, F16, F16, qkv=(q, k, v))
    major = [x.permute(1, 0, 2).contiguous().permute(1, 0, 2) for x in (q, k, v)]
    wide = torch.full((t, h * d + 64), 7.0, dtype=F16, device="cuda")
    L.attention_causal(ctx, *major, wide[:, :h * d], ints(cumulative(lens)), scale=d ** -0.5)
    ctx.sync()
    assert torch.equal(wide[:, :h * d].view(t, h, d), want)
    assert (wide[:, h * d:] == 7).all()


def test_causal_neighbours_do_not_leak(ctx):
    """NaN and infinities in one sequence leave the others as they were; a NaN key later in
    the same sequence leaves the rows before it."""
    lens, h, hk, d = [100, 60, 200], 4, 2, 128
    t = sum(lens)
    q, k, v = randn(1, t, h, d), randn(2, t, hk, d), randn(3, t, hk, d)
    clean = run_causal(ctx, lens, h, hk, d, BF16, BF16, qkv=(q, k, v))
    k[100:160] = math.nan
    v[100:160] = math.inf
    k[330] = math.nan
    o = torch.zeros_like(clean)
    L.attention_causal(ctx, q, k, v, o, ints(cumulative(lens)), scale=d ** -0.5)
    ctx.sync()
    keep = torch.ones(t, dtype=torch.bool)
    keep[100:160] = False
    keep[330:] = False
    assert torch.equal(o[keep.cuda()], clean[keep.cuda()])


@pytest.mark.parametrize("h,hk,d", [(128, 1, 64), (100, 1, 128), (65, 1, 64), (128, 2, 128)])
def test_causal_large_groups(ctx, h, hk, d):
    """One to two tokens per query tile, rows of the tile left over."""
    run_causal(ctx, [70, 3], h, hk, d, BF16, BF16, pad=1, seed=h)


def test_an_sm_budget_changes_no_result():
    own = L.Context(0)
    whole = run_causal(own, [900, 200], 16, 4, 128, BF16, BF16, seed=2)
    own.set_sm_budget(7)
    assert torch.equal(run_causal(own, [900, 200], 16, 4, 128, BF16, BF16, seed=2), whole)
    for q in (1, 90):
        Paged([q] * 5, [300, 2000, q, 700, 1500], 8, 2, 128, 32, BF16, seed=q).check(own)
    own.close()


def test_causal_same_bits_twice(ctx):
    a = run_causal(ctx, [700, 3, 250], 8, 2, 128, BF16, BF16, seed=1)
    b = run_causal(ctx, [700, 3, 250], 8, 2, 128, BF16, BF16, seed=1)
    assert torch.equal(a, b)


@pytest.mark.parametrize("cu", [[0, 50, 40, 60], [0, 10, 20, 1000], [-5, 10, 20, 30]])
def test_causal_bad_offsets_are_reported(ctx, cu):
    q, k, v = randn(1, 60, 4, 64), randn(2, 60, 2, 64), randn(3, 60, 2, 64)
    o = torch.zeros_like(q)
    L.attention_causal(ctx, q, k, v, o, ints(cu), scale=0.125)
    with pytest.raises(L.LlmrError) as e:
        ctx.sync()
    assert e.value.status == L.EINVAL
    ctx.sync()   # reported once


# -------------------------------------------------------------- paged attention

class Paged:
    """Requests over a cache whose unused rows and pages are NaN."""

    def __init__(self, q_lens, kv_lens, h, hk, d, page, dtype, *, pad=0, seed=0, size=1.0,
                 layout="dense", spare=3):
        self.q_lens, self.kv_list, self.d, self.dtype = q_lens, kv_lens, d, dtype
        need = [-(-x // page) for x in kv_lens]
        pages = sum(need) + spare
        shape = (pages, page, hk, d)
        if layout == "dense":
            kc, vc = (torch.full(shape, math.nan, dtype=dtype, device="cuda") for _ in range(2))
        elif layout == "together":      # K and V of a page side by side
            both = torch.full((pages, 2, page, hk, d), math.nan, dtype=dtype, device="cuda")
            kc, vc = both[:, 0], both[:, 1]
        else:                           # heads outside the rows of a page
            kc, vc = (torch.full((pages, hk, page, d), math.nan, dtype=dtype, device="cuda")
                      .permute(0, 2, 1, 3) for _ in range(2))
        order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
        table = torch.full((len(kv_lens), max(need + [1]) + 2), -1, dtype=torch.int32)
        self.k, self.v = [], []
        for i, n in enumerate(kv_lens):
            k = randn(seed + 10 * i + 1, n, hk, d, dtype=dtype, size=size)
            v = randn(seed + 10 * i + 2, n, hk, d, dtype=dtype)
            for c in range(need[i]):
                pg = order.pop()
                table[i, c] = pg
                part = slice(c * page, min(n, (c + 1) * page))
                kc[pg, :part.stop - part.start] = k[part]
                vc[pg, :part.stop - part.start] = v[part]
            self.k.append(k)
            self.v.append(v)
        t = sum(q_lens) + pad
        self.q = randn(seed + 7, t, h, d, dtype=dtype, size=size)
        self.kc, self.vc, self.table = kc, vc, table.cuda()
        self.cu, self.kv = ints(cumulative(q_lens)), ints(kv_lens)
        self.h, self.hk, self.t = h, hk, t

    def run(self, ctx, out_dtype=None, scale=None, max_q=None):
        scale = scale or self.d ** -0.5
        max_q = max_q or max(self.q_lens + [1])
        self.o = torch.full((self.t, self.h, self.d), 7.0, dtype=out_dtype or self.dtype, device="cuda")
        self.lse = torch.full((self.h, self.t), 7.0, device="cuda")
        ctx.reserve(L.attention_paged_workspace_bytes(
            n_seqs=len(self.q_lens), total_tokens=self.t, max_q_len=max_q, n_heads=self.h,
            n_kv_heads=self.hk, head_dim=self.d))
        L.attention_paged(ctx, self.q, self.kc, self.vc, self.o, self.cu, self.kv, self.table,
                          scale=scale, max_q_len=max_q, lse=self.lse)
        ctx.sync()
        return self.o

    def check(self, ctx, **kw):
        self.run(ctx, **kw)
        scale = kw.get("scale") or self.d ** -0.5
        at = 0
        for i, n in enumerate(self.q_lens):
            if n:
                rows = slice(at, at + n)
                w, wl, weight = R.rows_attention(self.q[rows], self.k[i], self.v[i], scale)
                vmax = float(self.v[i].abs().max()) if self.kv_list[i] else 0.0
                R.check_attention(self.o[rows], self.lse[:, rows], w, wl, weight, self.dtype, self.d,
                                  self.kv_list[i], vmax, R.score_size(self.q[rows], self.k[i], scale),
                                  (i, n, self.kv_list[i]))
            at += n
        assert (self.o[at:] == 7).all() and (self.lse[:, at:] == 7).all()
        return self.o


HEADS = [(4, 4, 64), (8, 2, 128), (14, 2, 64), (7, 1, 128), (32, 2, 64), (6, 2, 128)]


@pytest.mark.parametrize("h,hk,d", HEADS)
@pytest.mark.parametrize("page", [16, 64, 256])
def test_decode(ctx, h, hk, d, page):
    """One token each: contexts from nothing to several splits, a padded batch."""
    kv = [1, 17, 0, 128, 700, 129, 2500, 15]
    Paged([1] * len(kv), kv, h, hk, d, page, BF16, pad=2, seed=page).check(ctx)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("q_lens,kv_lens", [
    ([5, 1, 0, 3], [300, 40, 90, 3]),
    ([40, 7], [1000, 7]),
    ([129, 300], [129, 1111]),
])
def test_chunks(ctx, page, q_lens, kv_lens):
    Paged(q_lens, kv_lens, 8, 2, 128, page, BF16, pad=1, seed=page).check(ctx)


@pytest.mark.parametrize("h,hk,d", HEADS)
@pytest.mark.parametrize("q", [2, 3, 9, 33, 150])
def test_chunk_heads(ctx, h, hk, d, q):
    Paged([q, 1, q - 1], [1500, 260, q + 40], h, hk, d, 32, F16, seed=q).check(ctx)


@pytest.mark.parametrize("q", [1, 4, 20, 200])
def test_rows_without_a_key(ctx, q):
    """More queries than keys: the first rows see nothing and give 0 and -inf."""
    kv = [q // 2, 0, q, 600]
    p = Paged([q] * 4, kv, 8, 2, 128, 16, BF16, seed=q)
    p.check(ctx)
    assert (p.o[q:2 * q] == 0).all() and (p.lse[:, q:2 * q] == -math.inf).all()


@pytest.mark.parametrize("q", [1, 200])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("out_dtype", [F16, BF16, F32])
def test_paged_types(ctx, q, dtype, out_dtype):
    Paged([q, q], [333, 1200], 8, 2, 64, 16, dtype, seed=q).check(ctx, out_dtype=out_dtype)


@pytest.mark.parametrize("q", [1, 6, 100])
@pytest.mark.parametrize("layout", ["together", "heads"])
def test_cache_layouts(ctx, q, layout):
    Paged([q, q], [777, 90 + q], 8, 2, 128, 32, BF16, seed=q, layout=layout).check(ctx)


@pytest.mark.parametrize("q", [1, 130])
@pytest.mark.parametrize("h,hk,d", [(8, 1, 128), (4, 2, 64)])
def test_one_long_request(ctx, q, h, hk, d):
    """The long axis is split over the card and joined."""
    p = Paged([q], [20011], h, hk, d, 16, BF16, seed=2)
    a = p.check(ctx).clone()
    assert torch.equal(p.run(ctx), a)       # and joined in the same order every time


def test_peaked_and_growing_scores(ctx):
    for q in (1, 130):
        p = Paged([q], [3000], 8, 2, 128, 16, F16, seed=4)
        for at, f in ((500, 5), (1500, 10), (2900, 18)):
            p.k[0][at] *= f
            pg = int(p.table[0, at // 16])
            p.kc[pg, at % 16] *= f
        p.check(ctx)


@pytest.mark.parametrize("q", [1, 3, 8, 60, 200])
@pytest.mark.parametrize("kv", [1, 300, 9000])
def test_a_nan_key_is_seen(ctx, q, kv):
    """Rows that see a NaN key are NaN (and so is their LSE), also where it is the only one,
    and requests beside it are not."""
    kv = max(kv, q)
    p = Paged([q, q], [kv, kv], 8, 2, 128, 16, BF16, seed=q)
    at = kv - q                     # the first new token's own key: every row sees it
    p.kc[int(p.table[0, at // 16]), at % 16] = math.nan
    o = p.run(ctx).float()
    assert o[:q].isnan().all() and p.lse[:, :q].isnan().all()
    assert not o[q:].isnan().any() and not p.lse[:, q:].isnan().any()


def test_causal_nan_rows(ctx):
    q, k, v = randn(1, 300, 4, 64), randn(2, 300, 2, 64), randn(3, 300, 2, 64)
    k[0], k[150] = math.nan, math.nan
    o, lse = torch.zeros_like(q), torch.zeros((4, 300), device="cuda")
    L.attention_causal(ctx, q, k, v, o, ints([0, 100, 300]), scale=0.125, lse=lse)
    ctx.sync()
    bad = torch.zeros(300, dtype=torch.bool, device="cuda")
    bad[:100] = True
    bad[150:] = True
    assert o[bad].isnan().all() and lse[:, bad].isnan().all()
    assert not o[~bad].isnan().any() and not lse[:, ~bad].isnan().any()


def test_padded_bound_and_ragged_mix(ctx):
    """max_q_len above every request's rows; decodes and chunks in one call."""
    q = [1, 64, 1, 5, 0, 200, 1]
    kv = [900, 64, 1, 3000, 0, 1500, 129]
    Paged(q, kv, 16, 4, 128, 16, BF16, pad=5, seed=8).check(ctx, max_q=300)


def test_many_requests(ctx):
    g = torch.Generator().manual_seed(3)
    kv = torch.randint(0, 400, (700,), generator=g).tolist()
    Paged([1] * 700, kv, 4, 2, 64, 16, F16, seed=1).check(ctx)


def test_many_chunks(ctx):
    """More requests than a CTA scans at once, some without rows."""
    g = torch.Generator().manual_seed(4)
    kv = torch.randint(20, 300, (900,), generator=g).tolist()
    q = [17 * (i % 5 > 0) for i in range(900)]
    Paged(q, kv, 4, 2, 64, 16, F16, seed=1).check(ctx)


@pytest.mark.parametrize("q", [1, 3])
@pytest.mark.parametrize("h,hk", [(128, 1), (100, 1), (33, 1), (32, 1)])
def test_paged_large_groups(ctx, q, h, hk):
    Paged([q, q], [700, 90], h, hk, 64, 16, BF16, seed=q).check(ctx)


@pytest.mark.parametrize("q", [1, 100])
def test_two_contexts_at_once(q):
    """Calls of two contexts on two streams, each with its own workspace."""
    streams = [torch.cuda.Stream() for _ in range(2)]
    ctxs = [L.Context(0, stream=s) for s in streams]
    cases = [Paged([q] * 3, [3000, 900, 5000], 8, 2, 128, 16, BF16, seed=i) for i in range(2)]
    alone = [c.run(x).clone() for c, x in zip(cases, ctxs)]
    torch.cuda.synchronize()
    outs = [torch.zeros_like(a) for a in alone]
    torch.cuda.synchronize()
    for _ in range(20):
        for c, x, o in zip(cases, ctxs, outs):
            L.attention_paged(x, c.q, c.kc, c.vc, o, c.cu, c.kv, c.table, scale=c.d ** -0.5, max_q_len=q)
    for x in ctxs:
        x.sync()
    assert all(torch.equal(a, b) for a, b in zip(alone, outs))
    for x in ctxs:
        x.close()


def test_prompts_of_two_contexts_at_once():
    """Grids that take over their own units only, while both are on the GPU."""
    streams = [torch.cuda.Stream() for _ in range(2)]
    ctxs = [L.Context(0, stream=s) for s in streams]
    lens = [900, 30, 2000, 1, 1300]
    cases = [(randn(i, sum(lens), 16, 128), randn(i + 5, sum(lens), 4, 128), randn(i + 9, sum(lens), 4, 128))
             for i in range(2)]
    cu = ints(cumulative(lens))
    alone = [run_causal(x, lens, 16, 4, 128, BF16, BF16, qkv=c) for c, x in zip(cases, ctxs)]
    outs = [torch.zeros_like(a) for a in alone]
    torch.cuda.synchronize()
    for _ in range(20):
        for (q, k, v), x, o in zip(cases, ctxs, outs):
            L.attention_causal(x, q, k, v, o, cu, scale=128 ** -0.5)
    for x in ctxs:
        x.sync()
    assert all(torch.equal(a, b) for a, b in zip(alone, outs))
    for x in ctxs:
        x.close()


def test_captured_prompts_replay_with_other_lengths():
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        ctx = L.Context(0, stream=stream)
        t, h, hk, d = 3000, 8, 2, 64
        q, k, v = randn(1, t, h, d), randn(2, t, hk, d), randn(3, t, hk, d)
        o, cu = torch.zeros_like(q), ints([0, 1000, 1000, 2500])
        call = lambda: L.attention_causal(ctx, q, k, v, o, cu, scale=0.125)
        call()
        ctx.sync()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        call()
        call()
    with torch.cuda.stream(stream):
        for lens in ([3000, 0, 0], [1, 1, 1], [700, 1500, 300]):
            cu.copy_(ints(cumulative(lens)))
            o.fill_(7)
            g.replay()
            ctx.sync()
            got = o.clone()
            o.fill_(7)
            call()
            ctx.sync()
            assert torch.equal(got, o) and (o[sum(lens):] == 7).all()
    torch.cuda.synchronize()
    del g
    ctx.close()


def test_shared_pages(ctx):
    """Requests whose tables name the same pages (a common prefix)."""
    p = Paged([1, 1, 1], [640, 700, 666], 8, 2, 128, 64, BF16, seed=3)
    for i in (1, 2):
        p.table[i, :10] = p.table[0, :10]
        p.k[i][:640], p.v[i][:640] = p.k[0], p.v[0]
    p.check(ctx)
    p = Paged([50, 50], [640, 700], 8, 2, 128, 64, BF16, seed=3)
    p.table[1, :9] = p.table[0, :9]
    p.k[1][:576], p.v[1][:576] = p.k[0][:576], p.v[0][:576]
    p.check(ctx)


def test_cache_beyond_32_bit_offsets(ctx):
    """A cache of more than 2^31 elements: pages at its far end."""
    h, hk, d, page = 8, 8, 128, 256
    pages = (1 << 31) // (page * hk * d) + 9
    kc = torch.empty((pages, page, hk, d), dtype=F16, device="cuda")
    vc = torch.empty_like(kc)
    k, v = randn(1, 300, hk, d, dtype=F16), randn(2, 300, hk, d, dtype=F16)
    table = ints([[pages - 1, pages - 4]])
    for src, c in ((k, kc), (v, vc)):
        c[pages - 1] = src[:256]
        c[pages - 4, :44] = src[256:]
    for n in (1, 100):
        q = randn(3, n, h, d, dtype=F16)
        o = torch.zeros_like(q)
        ctx.reserve(L.attention_paged_workspace_bytes(n_seqs=1, total_tokens=n, max_q_len=n, n_heads=h,
                                                      n_kv_heads=hk, head_dim=d))
        L.attention_paged(ctx, q, kc, vc, o, ints([0, n]), ints([300]), table, scale=d ** -0.5,
                          max_q_len=n)
        ctx.sync()
        w, _, weight = R.rows_attention(q, k, v, d ** -0.5)
        R.check_attention(o, None, w, None, weight, F16, d, 300, float(v.abs().max()),
                          R.score_size(q, k, d ** -0.5))
    slots = ints([(pages - 1) * page + 7])
    L.paged_prologue(ctx, None, k[:1], v[:1], None, kc, vc, None, slots)
    ctx.sync()
    assert torch.equal(kc[pages - 1, 7], k[0]) and torch.equal(vc[pages - 1, 7], v[0])


@pytest.mark.parametrize("q,fault", [(130, "max_q")] + [
    (q, f) for q in (1, 130) for f in ("page_high", "page_low", "kv_long", "kv_negative", "cu")])
def test_bad_device_values_are_reported(ctx, q, fault):
    p = Paged([q, q], [500, 700], 8, 2, 128, 16, BF16, seed=1)
    max_q = q
    if fault == "page_high":
        p.table[0, 3] = p.kc.shape[0]
    elif fault == "page_low":
        p.table[0, 3] = -9
    elif fault == "kv_long":
        p.kv[0] = 1 << 20
    elif fault == "kv_negative":
        p.kv[0] = -4
    elif fault == "cu":
        p.cu[2] = 2 * q + 9
    else:
        max_q = q - 1
    with pytest.raises(L.LlmrError) as e:
        p.run(ctx, max_q=max_q)
    assert e.value.status == L.EINVAL
    good = Paged([q, q], [500, 700], 8, 2, 128, 16, BF16, seed=1)
    good.check(ctx)     # and the context goes on


# ------------------------------------------------------------------- planner

def run_plan(ctx, ctx_lens, new_lens, page, *, free_n=None, room=None, cols=None, inplace=False,
             seed=0, table_gap=0):
    held = [-(-c // page) for c in ctx_lens]
    last = [-(-(c + n) // page) for c, n in zip(ctx_lens, new_lens)]
    need = sum(last) - sum(held)
    free_n = need + 3 if free_n is None else free_n
    cols = cols or max(last + [1])
    n = len(ctx_lens)
    room = sum(new_lens) + 5 if room is None else room
    order = torch.randperm(sum(held) + free_n + 2, generator=torch.Generator().manual_seed(seed)).tolist()
    table = [[-1] * cols for _ in range(n)]
    for i, a in enumerate(held):
        for c in range(min(a, cols)):
            table[i][c] = order.pop()
    free = order[:free_n]
    dev_table = torch.full((n, cols + table_gap), -7, dtype=torch.int32)
    dev_table[:, :cols] = torch.tensor(table, dtype=torch.int32).view(n, cols)
    dev_table = dev_table.cuda()
    c, new, nf = ints(ctx_lens), ints(new_lens), ints([free_n])
    fp = ints(free + [99999])       # capacity beyond the stack's top
    fill = lambda k: torch.full((k,), -55, dtype=torch.int32, device="cuda")
    cu, pos, slots = fill(n + 1), fill(room), fill(room)
    kv, nfo = (c, nf) if inplace else (fill(n), fill(1))
    L.paged_plan(ctx, c, new, fp, nf, dev_table[:, :cols], cu, kv, pos, slots, nfo, page_size=page)
    got = lambda t: t.cpu().tolist()
    return (table, free), (lambda: (got(dev_table[:, :cols]), got(cu), got(kv), got(pos), got(slots),
                                    int(nfo))), dev_table


@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("ctx_lens,new_lens", [
    ([0], [1]), ([16, 15, 17, 0, 64], [1, 1, 1, 1, 1]), ([5, 0, 300], [0, 0, 0]),
    ([0, 100, 31, 0], [700, 0, 33, 5000]), ([], []),
])
def test_plan(ctx, page, inplace, ctx_lens, new_lens):
    (table, free), read, dev = run_plan(ctx, ctx_lens, new_lens, page, inplace=inplace, table_gap=3)
    ctx.sync()
    assert read() == R.plan(ctx_lens, new_lens, free, table, page, sum(new_lens) + 5)
    assert (dev[:, -3:] == -7).all()


@pytest.mark.parametrize("n", [33, 1025, 4096])
def test_plan_many_requests(ctx, n):
    g = torch.Generator().manual_seed(n)
    c = torch.randint(0, 200, (n,), generator=g).tolist()
    new = torch.randint(0, 12, (n,), generator=g).tolist()
    (table, free), read, _ = run_plan(ctx, c, new, 16, seed=n)
    ctx.sync()
    assert read() == R.plan(c, new, free, table, 16, sum(new) + 5)


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("what", ["pages", "tokens", "table", "negative", "huge"])
def test_plan_that_cannot_be_made_changes_nothing(ctx, what, inplace):
    c, new, kw = [40, 3, 16], [20, 50, 1], {}
    if what == "pages":
        kw["free_n"] = 4    # 5 are needed
    elif what == "tokens":
        kw["room"] = 70
    elif what == "table":
        kw["cols"] = 3
    elif what == "negative":
        c = [40, -3, 16]
        kw.update(cols=5, free_n=9)
    else:
        new = [2 ** 31 - 1, 2 ** 31 - 1, 1]
        kw.update(cols=5, free_n=9, room=80)
    (table, free), read, _ = run_plan(ctx, c, new, 16, inplace=inplace, **kw)
    with pytest.raises(L.LlmrError) as e:
        ctx.sync()
    assert e.value.status == (L.ENOMEM if what == "pages" else L.EINVAL)
    room = kw.get("room", 76)
    if what == "negative":
        room = 76
    assert read() == (table, [0] * 4, c, [0] * room, [-1] * room, len(free))


# ------------------------------------------------------------------ prologue

@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("in_dtype,dtype", [(BF16, BF16), (F16, F16), (F32, BF16), (BF16, F16)])
@pytest.mark.parametrize("tokens,h,hk,norm,rope", [(1, 8, 2, True, True), (37, 14, 2, True, True),
                                                   (130, 7, 7, False, True), (9, 40, 8, True, False),
                                                   (3, 1, 1, False, False)])
def test_prologue(ctx, d, half, in_dtype, dtype, tokens, h, hk, norm, rope):
    page, rows, eps = 16, 5000, 1e-6
    pages = -(-tokens // page) + 4
    g = torch.Generator().manual_seed(tokens)
    q, k, v = (randn(i, tokens, n, d, dtype=in_dtype) for i, n in ((1, h), (2, hk), (3, hk)))
    gains = [torch.rand(d, generator=g).cuda() * 0.4 + 0.8 for _ in range(2)]
    angle = torch.arange(rows)[:, None].double() * 10000.0 ** (-torch.arange(0, d, 2).double() / d)
    cos, sin = angle.cos().float().cuda(), angle.sin().float().cuda()
    pos = torch.randint(0, rows, (tokens,), generator=g).int().cuda()
    slots = torch.randperm(pages * page, generator=g)[:tokens].int().cuda()
    kc, vc = (torch.full((pages, page, hk, d), 7.0, dtype=dtype, device="cuda") for _ in range(2))
    q_out = torch.full((tokens, h, d), 7.0, dtype=dtype, device="cuda")
    if tokens > 4:
        slots[2] = -1       # padding
    L.paged_prologue(ctx, q, k, v, q_out, kc, vc, pos, slots, eps=eps,
                     q_gain=gains[0] if norm else None, k_gain=gains[1] if norm else None,
                     cos=cos if rope else None, sin=sin if rope else None, half=half and rope)
    ctx.sync()
    want = []
    for x, gain in ((q, gains[0]), (k, gains[1])):
        x = R.norm(x, gain, eps) if norm else x.double()
        want.append(R.rotate(x, cos[pos.long()], sin[pos.long()], half) if rope else x)
    live = slots >= 0
    at = slots[live].long()
    # The norm and the rotation in fp32: at most 16 roundings of values whose
    # size the row's largest bounds, the sum of D squares halved by the root;
    # then the output's own half step.
    def close(got, w):
        size = w.abs().amax(-1, keepdim=True)
        tol = w.abs() * R.half_step(dtype) + size * (16 + d / 2) * 2.0 ** -24 + 2.0 ** -25
        assert ((got.double() - w).abs() <= tol).all()
    close(q_out[live], want[0][live])
    close(kc.view(-1, hk, d)[at], want[1][live])
    assert torch.equal(vc.view(-1, hk, d)[at], v[live].to(dtype))
    rest = torch.ones(pages * page, dtype=torch.bool, device="cuda")
    rest[at] = False
    assert (kc.view(-1, hk, d)[rest] == 7).all() and (vc.view(-1, hk, d)[rest] == 7).all()
    assert (q_out[~live] == 7).all()


def test_prologue_in_place_and_strided(ctx):
    """q_out = q in a fused buffer, a cache with K and V side by side."""
    t, h, hk, d = 50, 6, 2, 128
    fused = randn(1, t, (h + 2 * hk) * d)
    keep = fused.clone()
    q, k, v = (x.unflatten(1, (-1, d)) for x in fused.split((h * d, hk * d, hk * d), 1))
    both = torch.zeros((4, 2, 16, hk, d), dtype=BF16, device="cuda")
    gain = torch.rand(d, device="cuda") + 0.5
    slots = ints(list(range(t))[::-1])
    plain = [torch.zeros((t, h, d), dtype=BF16, device="cuda"), torch.zeros_like(both[:, 0]),
             torch.zeros_like(both[:, 1])]
    L.paged_prologue(ctx, q, k, v, plain[0], plain[1], plain[2], None, slots, q_gain=gain)
    L.paged_prologue(ctx, q, k, v, q, both[:, 0], both[:, 1], None, slots, q_gain=gain)
    ctx.sync()
    assert torch.equal(q, plain[0]) and torch.equal(both[:, 0], plain[1])
    assert torch.equal(both[:, 1], plain[2]) and torch.equal(fused[:, h * d:], keep[:, h * d:])


@pytest.mark.parametrize("fault", ["slot", "position", "negative_position"])
def test_prologue_reports_bad_indices(ctx, fault):
    t, hk, d = 6, 2, 64
    k, v = randn(1, t, hk, d), randn(2, t, hk, d)
    kc, vc = (torch.zeros((2, 16, hk, d), dtype=BF16, device="cuda") for _ in range(2))
    cos = torch.ones((10, d // 2), device="cuda")
    sin = torch.zeros_like(cos)
    pos, slots = ints([0, 1, 2, 3, 4, 5]), ints([0, 1, 2, 3, 4, 5])
    if fault == "slot":
        slots[3] = 32
    elif fault == "position":
        pos[3] = 10
    else:
        pos[3] = -1
    L.paged_prologue(ctx, None, k, v, None, kc, vc, pos, slots, cos=cos, sin=sin)
    with pytest.raises(L.LlmrError) as e:
        ctx.sync()
    assert e.value.status == L.EINVAL
    good = [0, 1, 2, 4, 5]
    assert torch.equal(kc[0, good], k[good]) and (kc[0, 3] == 0).all() and (kc[1] == 0).all()


# ------------------------------------------------------------- as they are used

class Server:
    """Three requests served with the four operators; keeps every token's q, k, v."""

    def __init__(self, ctx, dtype=BF16, room=160):
        self.ctx, self.dtype, self.room = ctx, dtype, room
        self.n, self.h, self.hk, self.d, self.page = 3, 8, 2, 128, 16
        self.pages = 64
        z = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")
        self.lens, self.new, self.cu = z(self.n), z(self.n), z(self.n + 1)
        self.pos, self.slots = z(room), z(room)
        self.free = torch.randperm(self.pages, generator=torch.Generator().manual_seed(1)).int().cuda()
        self.n_free = ints([self.pages])
        self.table = torch.full((self.n, 20), -1, dtype=torch.int32, device="cuda")
        shape = (self.pages, self.page, self.hk, self.d)
        self.kc, self.vc = (torch.full(shape, math.nan, dtype=dtype, device="cuda") for _ in range(2))
        self.qkv = torch.zeros((room, (self.h + 2 * self.hk) * self.d), dtype=dtype, device="cuda")
        self.o = torch.zeros((room, self.h, self.d), dtype=dtype, device="cuda")
        angle = torch.arange(400)[:, None].double() * 10000.0 ** (-torch.arange(0, 128, 2).double() / 128)
        self.cos, self.sin = angle.cos().float().cuda(), angle.sin().float().cuda()
        self.gain = torch.rand(self.d, generator=torch.Generator().manual_seed(2)).cuda() + 0.5
        self.q_rot = torch.zeros((room, self.h, self.d), dtype=dtype, device="cuda")
        ctx.reserve(L.attention_paged_workspace_bytes(
            n_seqs=self.n, total_tokens=room, max_q_len=room, n_heads=self.h, n_kv_heads=self.hk,
            head_dim=self.d))

    def split(self):
        a, b = self.h * self.d, self.hk * self.d
        return (x.unflatten(1, (-1, self.d)) for x in self.qkv.split((a, b, b), 1))

    def step(self, max_q):
        q, k, v = self.split()
        L.paged_plan(self.ctx, self.lens, self.new, self.free, self.n_free, self.table, self.cu,
                     self.lens, self.pos, self.slots, self.n_free, page_size=self.page,
                     num_pages=self.pages)
        L.paged_prologue(self.ctx, q, k, v, self.q_rot, self.kc, self.vc, self.pos, self.slots,
                         q_gain=self.gain, k_gain=self.gain, cos=self.cos, sin=self.sin, half=True)
        L.attention_paged(self.ctx, self.q_rot, self.kc, self.vc, self.o, self.cu, self.lens,
                          self.table, scale=self.d ** -0.5, max_q_len=max_q)


STEPS = [[50, 0, 7], [1, 90, 1], [1, 1, 1], [30, 1, 0], [1, 1, 1], [1, 1, 1]]


def feed(server, i):
    server.new.copy_(torch.tensor(STEPS[i], dtype=torch.int32))
    server.qkv.copy_(randn(100 + i, *server.qkv.shape, dtype=server.dtype))


def whole_prompt(server, steps):
    """The same tokens as whole prompts through attention_causal, per request and step."""
    hist = [[[], [], []] for _ in range(server.n)]
    outs = []
    done = [0] * server.n
    for i in range(steps):
        feed(server, i)
        q, k, v = (x.clone() for x in server.split())
        at = 0
        rows = []
        for r, n in enumerate(STEPS[i]):
            pos = torch.arange(done[r], done[r] + n, device="cuda")
            for part, (x, turn) in enumerate(((q, True), (k, True), (v, False))):
                y = x[at:at + n]
                if turn:
                    y = R.norm(y, server.gain, 1e-6)
                    y = R.rotate(y, server.cos[pos], server.sin[pos], True).to(server.dtype)
                hist[r][part].append(y)
            rows.append((at, n))
            done[r] += n
            at += n
        qs, ks, vs = (torch.cat([torch.cat(hist[r][p]) for r in range(server.n)]) for p in range(3))
        o = torch.zeros_like(qs)
        L.attention_causal(server.ctx, qs, ks, vs, o, ints(cumulative(done)), scale=server.d ** -0.5)
        server.ctx.sync()
        ends = cumulative(done)
        outs.append([o[ends[r + 1] - n:ends[r + 1]] for r, (_, n) in enumerate(rows)])
    return outs


def compare_step(server, i, want):
    at = 0
    for r, n in enumerate(STEPS[i]):
        got = server.o[at:at + n].double()
        # Two kernels' roundings of the numerators (half a step each, beside
        # values of size ~|v| < 5) and of both outputs, and q or k rounded
        # the other way where the two norms' fp32 differ in the last place.
        tol = 4 * R.half_step(server.dtype) * 5
        assert ((got - want[r].double()).abs() <= tol).all(), (i, r)
        at += n


def test_serving_steps_equal_whole_prompts(ctx):
    s = Server(ctx)
    for i in range(len(STEPS)):
        feed(s, i)
        s.step(s.room)
        s.ctx.sync()
        got = s.o.clone()
        if i in (0, 1, 3, len(STEPS) - 1):
            keep = s.new.clone(), s.qkv.clone()
            want = whole_prompt(s, i + 1)[i]
            s.new.copy_(keep[0])
            s.qkv.copy_(keep[1])
        else:
            continue
        s.o.copy_(got)
        compare_step(s, i, want)
    used = [int(x) for x in s.lens]
    assert used == [sum(c) for c in zip(*STEPS)]
    assert int(s.n_free) == s.pages - sum(-(-u // s.page) for u in used)


@pytest.mark.parametrize("max_q", [1, 160])
def test_captured_step_replays(max_q):
    """One captured step (plan, prologue, attention) advances by itself and gives the eager bits."""
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        ctx = L.Context(0, stream=stream)
        eager, graphed = Server(ctx), Server(ctx)
        first = 0
        for s in (eager, graphed):
            feed(s, first)
            s.step(s.room)
        ctx.sync()
        for s in (eager, graphed):
            feed(s, 2)
        state = [x.clone() for x in (graphed.lens, graphed.n_free, graphed.table)]
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    n0 = ctx.launches
    with torch.cuda.graph(g, stream=stream):
        graphed.step(max_q)
    assert ctx.launches - n0 in (3, 4)   # attention joins its parts in a launch of its own
    with torch.cuda.stream(stream):
        for x, y in zip((graphed.lens, graphed.n_free, graphed.table), state):
            x.copy_(y)
        for i in (2, 4, 5):
            for s in (eager, graphed):
                feed(s, i)
            g.replay()
            eager.step(max_q)
            ctx.sync()
            assert torch.equal(eager.o, graphed.o) and torch.equal(eager.lens, graphed.lens)
            assert torch.equal(eager.table, graphed.table)
    torch.cuda.synchronize()
    del g
    ctx.close()


def test_other_stream(ctx):
    """A context on a stream of its own, inputs made on another and ordered by an event."""
    s = torch.cuda.Stream()
    own = L.Context(0, stream=s)
    q, k, v = randn(1, 300, 8, 64), randn(2, 300, 2, 64), randn(3, 300, 2, 64)
    o = torch.zeros_like(q)
    cu = ints([0, 300])
    s.wait_stream(torch.cuda.current_stream())
    L.attention_causal(own, q, k, v, o, cu, scale=0.125)
    own.sync()
    assert torch.equal(o, run_causal(ctx, [300], 8, 2, 64, BF16, BF16, qkv=(q, k, v)))
    own.close()


def test_refusals_of_the_library(ctx):
    """What the host can see is refused before anything is launched."""
    q, k, v = randn(1, 40, 4, 64), randn(2, 40, 2, 64), randn(3, 40, 2, 64)
    o, cu = torch.zeros_like(q), ints([0, 40])
    n0 = ctx.launches

    def refused(f, status=L.EINVAL):
        with pytest.raises(L.LlmrError) as e:
            f()
        assert e.value.status == status

    for bad in (0.0, -1.0, math.nan, math.inf):
        refused(lambda: L.attention_causal(ctx, q, k, v, o, cu, scale=bad))
    odd = torch.zeros(40 * 4 * 64 + 8, dtype=BF16, device="cuda")[1:-7].view(40, 4, 64)
    refused(lambda: L.attention_causal(ctx, odd, k, v, o, cu, scale=0.1))
    refused(lambda: L.attention_causal(ctx, q, k, v, odd, cu, scale=0.1))
    refused(lambda: L.attention_causal(ctx, q, k.cpu(), v, o, cu, scale=0.1))
    kc = torch.zeros((4, 24, 2, 64), dtype=BF16, device="cuda")      # page size
    table = ints([[0, 1]])
    refused(lambda: L.attention_paged(ctx, q, kc, kc, o, cu, ints([40]), table, scale=0.1, max_q_len=40))
    fresh = L.Context(0)
    kc = torch.zeros((4, 16, 2, 64), dtype=BF16, device="cuda")
    refused(lambda: L.attention_paged(fresh, q, kc, kc, o, cu, ints([32]), table, scale=0.1,
                                      max_q_len=40), L.ENOMEM)
    assert ctx.launches == n0 and fresh.launches == 0
    fresh.close()
    # Nothing to do is no error and launches nothing.
    e = lambda *s: torch.zeros(s, dtype=BF16, device="cuda")
    L.attention_causal(ctx, e(0, 4, 64), e(0, 2, 64), e(0, 2, 64), e(0, 4, 64), ints([0]), scale=0.1)
    assert ctx.launches == n0


def test_the_current_device_stays(ctx):
    before = torch.cuda.current_device()
    run_causal(ctx, [10], 4, 2, 64, BF16, BF16)
    assert torch.cuda.current_device() == before


# --------------------------------------------------------------- infinite scores

def check_infinite(o, lse, q, k, v, scale, dead, dtype, what):
    """Rows of one request whose first `dead` see scores of -inf alone: 0 / 0 and log 0."""
    w, wl, weight = R.rows_attention(q, k, v, scale)
    assert o[:dead].isnan().all() and (lse[:, :dead] == -math.inf).all(), what
    finite = k.clone()
    finite[..., 0] = finite[..., 0].nan_to_num(neginf=0.0)
    R.check_attention(o[dead:], lse[:, dead:], w[dead:], wl[:, dead:], weight[dead:], dtype, q.shape[2],
                      k.shape[0], float(v.abs().max()), R.score_size(q, finite, scale), what)


@pytest.mark.parametrize("q", [1, 4, 8, 20, 200])
@pytest.mark.parametrize("kv", [1, 300, 9000])
def test_rows_of_infinite_scores(ctx, q, kv):
    """Rows that see keys, each with a score of -inf, are no rows without a key."""
    kv, dead = max(kv, q), (q + 1) // 2
    p = Paged([q, q], [kv, kv], 8, 2, 128, 16, BF16, seed=q)
    p.q[:, :, 0] = p.q[:, :, 0].abs() + 0.5
    at = torch.arange(kv - q + dead, device="cuda")     # what the first `dead` rows see
    p.kc[p.table[0].long()[at // 16], at % 16, :, 0] = -math.inf
    p.k[0][at, :, 0] = -math.inf
    o, scale = p.run(ctx), p.d ** -0.5
    check_infinite(o[:q], p.lse[:, :q], p.q[:q], p.k[0], p.v[0], scale, dead, BF16, (q, kv))
    check_infinite(o[q:], p.lse[:, q:], p.q[q:], p.k[1], p.v[1], scale, 0, BF16, (q, kv))


@pytest.mark.parametrize("h,hk,d", [(8, 2, 128), (14, 2, 64), (32, 8, 128)])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("lens", [[100, 700, 3], [5000]])
def test_causal_rows_of_infinite_scores(ctx, h, hk, d, dtype, lens):
    t = sum(lens)
    q, k, v = (randn(i, t, n, d, dtype=dtype) for i, n in ((1, h), (2, hk), (3, hk)))
    q[:, :, 0] = q[:, :, 0].abs() + 0.5
    dead = [2 * n // 5 for n in lens]
    cu = cumulative(lens)
    for at, x in zip(cu, dead):
        k[at:at + x, :, 0] = -math.inf
    o, lse = torch.zeros_like(q), torch.zeros((h, t), device="cuda")
    L.attention_causal(ctx, q, k, v, o, ints(cu), scale=d ** -0.5, lse=lse)
    ctx.sync()
    for at, n, x in zip(cu, lens, dead):
        part = slice(at, at + n)
        check_infinite(o[part], lse[:, part], q[part], k[part], v[part], d ** -0.5, x, dtype, (lens, at))


# ------------------------------------------------- bad offsets beside good requests

# Offsets, tokens, and the sequences that stay right: in order and in range themselves,
# behind the earlier ones, and in no row that another ascending pair of offsets claims.
BAD_OFFSETS = [([0, 1000, 0, 0], 1000, [0]), ([0, 1000, -1, 2000], 2000, [0]),
               ([0, 100, 9999, 400, 700], 700, [0, 3]), ([-5, 300, 1200, 1200, 1300], 1300, [1, 3]),
               ([0, 500, 400, 2 ** 31 - 1, 900, 1500], 1500, [0, 4]),
               ([700, 1500, -2 ** 31, 0, 650], 1500, [0]), ([0, 300, 250, 260, 900, 1500], 1500, [4]),
               ([2 ** 31 - 1] * 40 + [0, 333, 1000], 1000, [40, 41])]


@pytest.mark.parametrize("cu,tokens,good", BAD_OFFSETS)
@pytest.mark.parametrize("h,hk,d", [(4, 2, 64), (14, 2, 64), (32, 8, 128), (8, 8, 128)])
@pytest.mark.parametrize("budget", [0, 5])
def test_bad_offsets_leave_other_sequences(cu, tokens, good, h, hk, d, budget):
    own = L.Context(0)
    own.set_sm_budget(budget)
    q, k, v = (randn(i, tokens, n, d) for i, n in ((1, h), (2, hk), (3, hk)))
    o, lse = torch.full_like(q, 7.0), torch.full((h, tokens), 7.0, device="cuda")
    torch.cuda.synchronize()
    L.attention_causal(own, q, k, v, o, ints(cu), scale=d ** -0.5, lse=lse)
    with pytest.raises(L.LlmrError) as e:
        own.sync()
    assert e.value.status == L.EINVAL
    for i in good:
        part = slice(cu[i], cu[i + 1])
        w, wl, weight = R.rows_attention(q[part], k[part], v[part], d ** -0.5)
        R.check_attention(o[part], lse[:, part], w, wl, weight, BF16, d, cu[i + 1] - cu[i],
                          float(v[part].abs().max()), R.score_size(q[part], k[part], d ** -0.5), (cu, i))
    own.close()


@pytest.mark.parametrize("big", [False, True])
def test_bad_offsets_among_many_sequences(ctx, big):
    """Bad values here and there between hundreds of sequences, some of them long."""
    g = torch.Generator().manual_seed(11)
    lens = torch.randint(0, 90 if big else 9, (900,), generator=g).tolist()
    lens[300] = 1500
    cu, tokens = cumulative(lens), sum(lens)
    for at, x in ((0, -1), (17, 2 ** 30), (299, -7), (400, 0), (401, tokens + 1), (650, -2 ** 31), (900, -2)):
        cu[at] = x
    h, hk, d = 8, 2, 64
    q, k, v = (randn(i, tokens, n, d, dtype=F16) for i, n in ((1, h), (2, hk), (3, hk)))
    o = torch.full_like(q, 7.0)
    L.attention_causal(ctx, q, k, v, o, ints(cu), scale=0.125)
    with pytest.raises(L.LlmrError):
        ctx.sync()
    for i, (a, b) in enumerate(zip(cu, cu[1:])):
        if 0 <= a < b <= tokens:
            part = slice(a, b)
            w, _, weight = R.rows_attention(q[part], k[part], v[part], 0.125)
            R.check_attention(o[part], None, w, None, weight, F16, d, b - a, float(v[part].abs().max()),
                              R.score_size(q[part], k[part], 0.125), i)


def test_captured_prompts_report_bad_offsets_and_recover():
    """A replay with bad offsets, then one with good ones: the verdict belongs to its launch."""
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        own = L.Context(0, stream=stream)
        t, h, hk, d = 3000, 16, 4, 64
        q, k, v = randn(1, t, h, d), randn(2, t, hk, d), randn(3, t, hk, d)
        o, cu = torch.zeros_like(q), ints([0, 1000, 1800, 3000])
        call = lambda: L.attention_causal(own, q, k, v, o, cu, scale=0.125)
        call()
        own.sync()
        want = o.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        call()
    with torch.cuda.stream(stream):
        for bad in ([0, 1000, -1, 3000], [0, 1000, 1 << 30, 3000]):
            cu.copy_(ints(bad))
            o.fill_(7)
            g.replay()
            with pytest.raises(L.LlmrError):
                own.sync()
            assert torch.equal(o[:1000], want[:1000])
            cu.copy_(ints([0, 1000, 1800, 3000]))
            o.fill_(7)
            g.replay()
            own.sync()
            assert torch.equal(o, want)
    torch.cuda.synchronize()
    del g
    own.close()


@pytest.mark.parametrize("q", [1, 5, 130])
@pytest.mark.parametrize("fault", ["page_high", "page_low", "kv_long", "kv_negative", "cu_high", "cu_low", "rows"])
def test_bad_requests_leave_the_others(ctx, q, fault):
    """Five requests, the third (with bad offsets its neighbour too) at fault."""
    p = Paged([q] * 5, [500, 2700, 900, 3000, q], 8, 2, 128, 16, BF16, seed=1)
    kw, concerned = {}, [2]
    if fault.startswith("page"):
        p.table[2, 3] = p.kc.shape[0] if fault == "page_high" else -9
    elif fault.startswith("kv"):
        p.kv[2] = 1 << 20 if fault == "kv_long" else -4
    elif fault.startswith("cu"):
        p.cu[3] = 99 * q if fault == "cu_high" else -3
        concerned = [2, 3]
    else:    # more rows than max_q_len allows
        p = Paged([q, q, q + 1, q, q], [500, 2700, 900, 3000, q], 8, 2, 128, 16, BF16, seed=1)
        kw["max_q"] = q
    with pytest.raises(L.LlmrError) as e:
        p.run(ctx, **kw)
    assert e.value.status == L.EINVAL
    at = 0
    for i, n in enumerate(p.q_lens):
        if i not in concerned:
            rows = slice(at, at + n)
            w, wl, weight = R.rows_attention(p.q[rows], p.k[i], p.v[i], p.d ** -0.5)
            R.check_attention(p.o[rows], p.lse[:, rows], w, wl, weight, BF16, p.d, p.kv_list[i],
                              float(p.v[i].abs().max()), R.score_size(p.q[rows], p.k[i], p.d ** -0.5), (fault, i))
        at += n


def test_bad_offsets_in_two_contexts_at_once():
    """Where another grid holds SMs, CTAs take over units of the first of their grid."""
    streams = [torch.cuda.Stream() for _ in range(2)]
    ctxs = [L.Context(0, stream=s) for s in streams]
    t, cu = 6000, ints([0, 1700, -3, 2500, 4200, 9999, 4300, 6000])
    good = [slice(0, 1700), slice(2500, 4200), slice(4300, 6000)]
    cases = [(randn(i, t, 16, 128), randn(i + 5, t, 4, 128), randn(i + 9, t, 4, 128)) for i in range(2)]
    torch.cuda.synchronize()
    want = []
    for (q, k, v), x in zip(cases, ctxs):
        alone = torch.zeros_like(q)
        torch.cuda.synchronize()
        L.attention_causal(x, q, k, v, alone, ints([0, 1700, 2500, 4200, 4300, 6000]), scale=128 ** -0.5)
        x.sync()
        want.append(alone)
    outs = [[torch.zeros_like(a) for _ in range(10)] for a in want]
    torch.cuda.synchronize()
    for r in range(10):
        for (q, k, v), x, o in zip(cases, ctxs, outs):
            L.attention_causal(x, q, k, v, o[r], cu, scale=128 ** -0.5)
    for x in ctxs:
        with pytest.raises(L.LlmrError):
            x.sync()
    assert all(torch.equal(o[part], w[part]) for w, os in zip(want, outs) for o in os for part in good)
    for x in ctxs:
        x.close()


# -------------------------------------------------- more than one error before a sync

def statuses(ctx):
    out = []
    for _ in range(4):
        try:
            ctx.sync()
            return out
        except L.LlmrError as e:
            out.append(e.status)
    return out


@pytest.mark.parametrize("pages_first", [False, True])
@pytest.mark.parametrize("timeout", [False, True])
def test_sync_reports_every_condition(ctx, pages_first, timeout):
    """A bad slot and a step without pages between two syncs: neither hides the other."""
    k, v = randn(1, 3, 2, 64), randn(2, 3, 2, 64)
    kc, vc = (torch.zeros((2, 16, 2, 64), dtype=BF16, device="cuda") for _ in range(2))

    def bad_slot():
        L.paged_prologue(ctx, None, k, v, None, kc, vc, None, ints([0, 32, 5]))

    plans = []

    def no_pages():
        plans.append(run_plan(ctx, [40, 3], [20, 50], 16, free_n=2))

    calls = [no_pages, bad_slot] if pages_first else [bad_slot, no_pages]
    if timeout:
        calls.insert(1, lambda: ctx.check(L.lib.llmr_selftest_wait_timeout(ctx.handle, 20_000_000)))
    for f in calls:
        f()
    assert statuses(ctx) == [L.ETIMEOUT] * timeout + [L.ENOMEM, L.EINVAL]
    assert plans[0][1]()[1] == [0, 0, 0]        # cu_q: nothing was planned
    assert torch.equal(kc[0, [0, 5]], k[[0, 2]])
    bad_slot()
    bad_slot()
    assert statuses(ctx) == [L.EINVAL]


# ------------------------------------------------------------------- the SM budget

def captured_kernels(stream, call):
    """(name, CTAs) of the kernels that a call launches, from a capture of it."""
    from cuda.bindings import driver
    g = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(g, stream=stream):
        call()
    graph = driver.CUgraph(int(g.raw_cuda_graph()))
    _, _, n = driver.cuGraphGetNodes(graph)
    _, nodes, n = driver.cuGraphGetNodes(graph, n)
    out = []
    for node in nodes:
        err, p = driver.cuGraphKernelNodeGetParams(node)
        assert err == driver.CUresult.CUDA_SUCCESS
        err, name = driver.cuFuncGetName(p.func)
        assert err == driver.CUresult.CUDA_SUCCESS
        out.append((name.decode(), p.gridDimX * p.gridDimY * p.gridDimZ))
    return out


@pytest.mark.parametrize("budget", [1, 7, 40, 100])
@pytest.mark.parametrize("q", [1, 4, 8, 90])
def test_attention_keeps_to_the_sm_budget(budget, q):
    """A CTA per SM of the budget: CTAs go to free SMs first, also where two fit one SM."""
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        own = L.Context(0, stream=stream)
        own.set_sm_budget(budget)
        p = Paged([q] * 40, [300, 2000, q, 700, 1500] * 8, 8, 2, 128, 32, BF16, seed=q)
        p.check(own)
        cu = ints([0, 15 * q, 40 * q])
        k, v = randn(1, p.t, 2, 128), randn(2, p.t, 2, 128)
    torch.cuda.synchronize()
    paged = captured_kernels(stream, lambda: L.attention_paged(
        own, p.q, p.kc, p.vc, p.o, p.cu, p.kv, p.table, scale=0.1, max_q_len=q))
    causal = captured_kernels(stream, lambda: L.attention_causal(own, p.q, k, v, p.o, cu, scale=0.1))
    seen = [(n, ctas) for n, ctas in paged + causal if "join" not in n]
    assert len(seen) == 2 and all(ctas <= budget for _, ctas in seen), seen
    own.close()


# ------------------------------------------------------------- joins of large scores

@pytest.mark.parametrize("q", [1, 8, 20, 130])
@pytest.mark.parametrize("kv", [3001, 9000, 20011])
@pytest.mark.parametrize("d", [64, 128])
def test_joins_of_large_scores(ctx, q, kv, d):
    """Every score is 30720, so all keys weigh the same, and V is 1 in the first half and -1 in
    the second: what the parts of a split row weigh against one another shows alone."""
    p = Paged([q], [kv], 8, 2, d, 16, F16, seed=3)
    p.q.zero_()
    p.q[..., 0] = 256
    for x, c in ((p.kc, p.k), (p.vc, p.v)):
        x.zero_()
        c[0].zero_()
    p.kc[..., 0] = 120
    p.k[0][..., 0] = 120
    p.v[0][:kv // 2] = 1
    p.v[0][kv // 2:] = -1
    at = torch.arange(kv, device="cuda")
    p.vc[p.table[0].long()[at // 16], at % 16] = p.v[0]
    o = p.run(ctx, out_dtype=F32, scale=1.0).double()
    w, wl, _ = R.rows_attention(p.q, p.k[0], p.v[0], 1.0)
    # The numerators are one value c 2^e of 11 bits, and O sums +-1 of them: exact (below
    # 2^24 steps). l adds 32 of them at a time in fp32, then 4 such sums, then blocks of
    # 128 keys: 40 + kv / 64 roundings at most, parts included. The rounding of c itself is
    # common to all keys, half a step of o.
    tol = (40 + kv / 64) * 2.0 ** -24 + w.abs() * R.half_step(F16)
    assert ((o - w).abs() <= tol).all(), ((o - w).abs() / tol).max().item()
    assert ((p.lse.double() - wl).abs() <= 2.0 ** -23 * wl).all()


# ------------------------------------------------------- large plans, four places a thread

def check_large_plan(ctx, ctx_lens, new_lens, page, room, shift, inplace=False):
    """A plan whose positions and slots begin `shift` elements behind a 16-byte boundary."""
    held = [-(-c // page) for c in ctx_lens]
    last = [-(-(c + n) // page) for c, n in zip(ctx_lens, new_lens)]
    need, n = sum(last) - sum(held), len(ctx_lens)
    order = torch.randperm(sum(held) + need + 9, generator=torch.Generator().manual_seed(room)).tolist()
    table, at = [], 0
    for a in held:
        table.append(order[at:at + a] + [-1] * (max(last) - a))
        at += a
    free = order[at:]
    dev, c, nf, fp = ints(table), ints(ctx_lens), ints([len(free)]), ints(free)
    pos, slots = (torch.full((room + 8,), -55, dtype=torch.int32, device="cuda") for _ in range(2))
    cu = torch.full((n + 1,), -55, dtype=torch.int32, device="cuda")
    kv, nfo = (c, nf) if inplace else (torch.zeros_like(c), torch.zeros_like(nf))
    L.paged_plan(ctx, c, ints(new_lens), fp, nf, dev, cu, kv, pos[shift:shift + room], slots[shift:shift + room],
                 nfo, page_size=page, num_pages=len(order))
    ctx.sync()
    want = R.plan(ctx_lens, new_lens, free, table, page, room)
    got = [x.cpu().tolist() for x in (dev, cu, kv, pos[shift:shift + room], slots[shift:shift + room])]
    assert (*got, int(nfo)) == want
    for x in (pos, slots):      # nothing beside the arrays
        assert (x[:shift] == -55).all() and (x[shift + room:] == -55).all()


@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("over", [0, 1, 2, 3])
@pytest.mark.parametrize("shift", [0, 1, 2, 3])
def test_large_plan(ctx, page, over, shift):
    """More than 32768 places: four of a thread across requests' borders, a ragged end."""
    g = torch.Generator().manual_seed(4 * over + shift)
    new = [0, 1, 1, 1, 0, 0, 2, 1, 9000, 0, 3, 1, 1, 20000, 5, 0, 1] + torch.randint(0, 3, (600,), generator=g).tolist()
    new += [4001 - shift, 0, 0]
    ctx_lens = torch.randint(0, 300, (len(new),), generator=g).tolist()
    ctx_lens[8], ctx_lens[13] = page, page - 1
    room = (max(sum(new), 32768) + 4) // 4 * 4 + 4 + over
    check_large_plan(ctx, ctx_lens, new, page, room, shift, inplace=over == 1)


@pytest.mark.parametrize("shift", [0, 1])
def test_large_plan_that_fills_its_places(ctx, shift):
    """No place behind the last token, and one request alone."""
    for total in (32769, 40002, 65536):
        check_large_plan(ctx, [77], [total], 64, total, shift)
        check_large_plan(ctx, [3] * (total // 8) if total // 8 <= 4096 else [3] * 4096,
                         [8] * min(total // 8, 4096), 16, max(total, 32769), shift)


def test_large_plan_reports_a_bad_page(ctx):
    """One table entry and one free page out of range: their tokens get no slot, the others do."""
    page, c, new = 64, [100, 0, 200], [30000, 100, 9000]
    held = [2, 0, 4]
    need = [-(-30100 // page) - 2, 2, -(-9200 // page) - 4]
    order = list(range(sum(held) + sum(need)))
    table = [order[:2] + [-1] * (need[0] + 2), [-1] * (need[0] + 4), order[2:6] + [-1] * need[0]]
    free = order[6:]
    bad_free = len(free) - 1 - (need[0] + 1)      # the second request's second page
    free[bad_free] = 1 << 20
    table[2][3] = -4                              # where the third's tokens begin
    room = sum(new) + 5
    dev, cu, kv, pos, slots, nfo = (ints(x) for x in (table, [0] * 4, [0] * 3, [0] * room, [0] * room, [0]))
    L.paged_plan(ctx, ints(c), ints(new), ints(free), ints([len(free)]), dev, cu, kv, pos, slots, nfo,
                 page_size=page, num_pages=len(order))
    assert statuses(ctx) == [L.EINVAL]
    want = R.plan(c, new, free, table, page, room)
    slot = [s if 0 <= s < len(order) * page else -1 for s in want[4]]
    assert slots.tolist() == slot and slot.count(-1) == 5 + (100 - 64) + (256 - 200)
    assert pos.tolist() == want[3] and cu.tolist() == want[1]


# ------------------------------------------- which V a split row meets, block by block

def paged_v(p, i, kv, v):
    """Puts v [kv, heads, D] into request i's pages."""
    at = torch.arange(kv, device="cuda")
    page = p.vc.shape[1]
    p.vc[p.table[i].long()[at // page], at % page] = v


@pytest.mark.parametrize("q", [1, 8, 20, 130])
@pytest.mark.parametrize("h,hk,d", [(8, 2, 128), (4, 1, 64)])
def test_every_block_of_v_counts(ctx, q, h, hk, d):
    """V is zero but for 64 keys at a time, so a block that is lost, doubled or swapped at a border
    of a range, a page or a tile is the whole result."""
    kv = 20011
    p = Paged([q], [kv], h, hk, d, 16, BF16, seed=5)
    x = torch.einsum("nhd,mhd->hnm", p.q.double(), p.k[0].double().repeat_interleave(h // hk, 1)) * d ** -0.5
    at = torch.arange(kv, device="cuda")
    x = x.masked_fill(at[None] > kv - q + torch.arange(q, device="cuda")[:, None], -math.inf)
    prob = torch.softmax(x, -1)
    v = p.v[0].clone()
    smax = R.score_size(p.q, p.k[0], d ** -0.5)
    worst = 0.0
    for b in range(0, kv, 64):
        part = slice(b, min(b + 64, kv))
        one = torch.zeros_like(v)
        one[part] = v[part]
        paged_v(p, 0, kv, one)
        o = p.run(ctx).double()
        wide = v[part].double().repeat_interleave(h // hk, 1)
        w, weight = (torch.einsum("hnm,mhd->nhd", prob[..., part], y) for y in (wide, wide.abs()))
        bound = R.attention_bound(w, weight, BF16, BF16, d, kv, float(v.abs().max()), smax)
        worst = max(worst, ((o - w).abs() / bound).max().item())
        assert worst <= 1, (b, worst)
        assert bound[-1].mean() < 0.05 * weight[-1].mean()    # (a lost block would show)


@pytest.mark.parametrize("q", [1, 5, 60])
def test_every_block_of_v_counts_in_a_batch(ctx, q):
    """The same over many requests: V of every seventh block of 64 keys, in turn."""
    kv = [700, 5000, 64, 8191, 2, 129, 3000, 6000, 300, 4097]
    kv = [max(q, n) for n in kv]
    p = Paged([q] * len(kv), kv, 8, 2, 128, 32, BF16, seed=6)
    full = [v.clone() for v in p.v]
    for turn in range(7):
        for i, n in enumerate(kv):
            keep = (torch.arange(n, device="cuda") // 64 % 7 == turn)[:, None, None]
            p.v[i] = torch.where(keep, full[i], 0)
            paged_v(p, i, n, p.v[i])
        p.check(ctx)


# ------------------------------------------------------------------- strided paged calls

@pytest.mark.parametrize("q", [1, 4, 8, 90])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("out_dtype", [BF16, F32])
def test_paged_strides(ctx, q, d, out_dtype):
    """q inside a fused projection and head-major, o with gaps, with heads outside and flat, and a
    block table that is part of a wider one."""
    h, hk = 8, 2
    p = Paged([q, 0, q + 1, q], [700, 40, 3000, q], h, hk, d, 16, BF16, pad=2, seed=q)
    want = p.check(ctx, out_dtype=out_dtype).clone()
    want_lse = p.lse.clone()
    fused = randn(9, p.t, (h + 2 * hk) * d)
    fused[:, :h * d] = p.q.flatten(1)
    major = p.q.transpose(0, 1).contiguous().transpose(0, 1)
    spread = torch.zeros((p.t, h, d + 64), dtype=BF16, device="cuda")
    spread[..., :d] = p.q
    wide_table = torch.full((4, p.table.shape[1] + 9), 1 << 20, dtype=torch.int32, device="cuda")
    cols = slice(3, 3 + p.table.shape[1])
    wide_table[:, cols] = p.table
    for query in (fused[:, :h * d].unflatten(1, (h, d)), major, spread[..., :d]):
        flat = torch.full((p.t, h * d + 64), 7.0, dtype=out_dtype, device="cuda")
        outer = torch.full((h, p.t, d), 7.0, dtype=out_dtype, device="cuda")
        gaps = torch.full((p.t, h, d + 64), 7.0, dtype=out_dtype, device="cuda")
        for o, got in ((flat[:, :h * d], flat[:, :h * d].unflatten(1, (h, d))),
                       (outer.transpose(0, 1), outer.transpose(0, 1)), (gaps[..., :d], gaps[..., :d])):
            lse = torch.full((h, p.t), 7.0, device="cuda")
            L.attention_paged(ctx, query, p.kc, p.vc, o, p.cu, p.kv, wide_table[:, cols], scale=d ** -0.5,
                              max_q_len=q + 1, lse=lse)
            ctx.sync()
            assert torch.equal(got, want) and torch.equal(lse, want_lse)
        assert (flat[:, h * d:] == 7).all() and (gaps[..., d:] == 7).all()


# ------------------------------------------------- a prompt that is not cached, both steps

@pytest.mark.parametrize("h,hk,d,half", [(8, 2, 128, True), (14, 2, 64, False)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_uncached_prompts_norm_rope_and_attention(ctx, h, hk, d, half, dtype):
    """Norm + RoPE into dense q and k: the prologue with slots 0 .. tokens - 1 and dense buffers as a
    cache, which attention_causal then reads."""
    lens, page = [77, 1, 300, 45], 16
    t = sum(lens)
    rows = -(-t // page) * page
    fused = randn(1, t, (h + 2 * hk) * d, dtype=dtype)
    q, k, v = (x.unflatten(1, (-1, d)) for x in fused.split((h * d, hk * d, hk * d), 1))
    angle = torch.arange(400)[:, None].double() * 10000.0 ** (-torch.arange(0, d, 2).double() / d)
    cos, sin = angle.cos().float().cuda(), angle.sin().float().cuda()
    gains = [torch.rand(d, generator=torch.Generator().manual_seed(i)).cuda() + 0.5 for i in range(2)]
    pos = torch.cat([torch.arange(n) for n in lens]).int().cuda()
    slots = torch.arange(t, dtype=torch.int32, device="cuda")
    q_rot = torch.zeros((t, h, d), dtype=dtype, device="cuda")
    k_rot, v_rot = (torch.zeros((rows, hk, d), dtype=dtype, device="cuda") for _ in range(2))
    L.paged_prologue(ctx, q, k, v, q_rot, k_rot.view(-1, page, hk, d), v_rot.view(-1, page, hk, d), pos, slots,
                     q_gain=gains[0], k_gain=gains[1], cos=cos, sin=sin, half=half)
    o = torch.zeros_like(q_rot)
    L.attention_causal(ctx, q_rot, k_rot[:t], v_rot[:t], o, ints(cumulative(lens)), scale=d ** -0.5)
    ctx.sync()
    for x, gain, got in ((q, gains[0], q_rot), (k, gains[1], k_rot[:t])):
        w = R.rotate(R.norm(x, gain, 1e-6), cos[pos.long()], sin[pos.long()], half)
        size = w.abs().amax(-1, keepdim=True)
        tol = w.abs() * R.half_step(dtype) + size * (16 + d / 2) * 2.0 ** -24 + 2.0 ** -25
        assert ((got.double() - w).abs() <= tol).all()
    assert torch.equal(v_rot[:t], v)
    at = 0
    for n in lens:
        part = slice(at, at + n)
        w, _, weight = R.rows_attention(q_rot[part], k_rot[part], v[part], d ** -0.5)
        R.check_attention(o[part], None, w, None, weight, dtype, d, n, float(v[part].abs().max()),
                          R.score_size(q_rot[part], k_rot[part], d ** -0.5), at)
        at += n


# ------------------------------------------- overlapped starts behind other kinds of work

@pytest.mark.parametrize("max_q", [1, 160])
@pytest.mark.parametrize("captured", [False, True])
def test_steps_wait_for_copies_and_other_streams(max_q, captured):
    """A step's kernels start while the one before ends; here that is a copy, a memset, or a wait for
    late work of another stream, between calls of the library and in a capture."""
    main, side = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(main):
        ctx = L.Context(0, stream=main)
        plain, mixed = Server(ctx), Server(ctx)
        for s in (plain, mixed):
            feed(s, 0)
            s.step(s.room)
        ctx.sync()
        late_new, late_qkv = torch.zeros_like(mixed.new), torch.zeros_like(mixed.qkv)
        late_lens = torch.zeros_like(mixed.lens)

    def step():
        # Behind library kernels (the step before): a memset, then inputs that another stream makes late.
        mixed.o.zero_()
        fork = torch.cuda.Event()
        fork.record(main)
        with torch.cuda.stream(side):
            side.wait_event(fork)
            torch.cuda._sleep(2_000_000)
            mixed.new.copy_(late_new)
            mixed.qkv.copy_(late_qkv)
            join = torch.cuda.Event()
            join.record(side)
        main.wait_event(join)
        mixed.step(max_q)
        # A copy between two library kernels: its target is the next call's input.
        mixed.lens.add_(1)
        mixed.lens.sub_(1)
        late_lens.copy_(mixed.lens)

    with torch.cuda.stream(main):
        if captured:
            state = [x.clone() for x in (mixed.lens, mixed.n_free, mixed.table)]
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=main):
                step()
            for x, y in zip((mixed.lens, mixed.n_free, mixed.table), state):
                x.copy_(y)
        for i in (2, 4, 5):
            feed(plain, i)
            late_new.copy_(plain.new)
            late_qkv.copy_(plain.qkv)
            plain.o.zero_()
            plain.step(max_q)
            g.replay() if captured else step()
            ctx.sync()
            assert torch.equal(plain.o, mixed.o) and torch.equal(plain.lens, mixed.lens)
            assert torch.equal(plain.table, mixed.table) and torch.equal(late_lens, mixed.lens)
    torch.cuda.synchronize()
    if captured:
        del g
    ctx.close()


def test_prompts_and_paged_calls_in_turn(ctx):
    """Grids with and without an overlapped start behind one another, each reading what the one before
    wrote: prologue, prompts, a paged call over the same keys."""
    h, hk, d, t = 8, 2, 128, 300
    q, k, v = (randn(i, t, n, d) for i, n in ((1, h), (2, hk), (3, hk)))
    gain = torch.rand(d, generator=torch.Generator().manual_seed(1)).cuda() + 0.5
    rows = 304
    table = torch.arange(rows // 16, dtype=torch.int32, device="cuda").view(1, -1)
    slots, cu, lens = torch.arange(t, dtype=torch.int32, device="cuda"), ints([0, t]), ints([t])
    ctx.reserve(L.attention_paged_workspace_bytes(n_seqs=1, total_tokens=t, max_q_len=t, n_heads=h,
                                                  n_kv_heads=hk, head_dim=d))
    first = None
    for turn in range(12):
        q_rot = torch.full_like(q, math.nan)
        kc, vc = (torch.full((rows // 16, 16, hk, d), math.nan, dtype=BF16, device="cuda") for _ in range(2))
        a, b, c = (torch.full_like(q, math.nan) for _ in range(3))
        for o in (a, c):
            L.paged_prologue(ctx, q, k, v, q_rot, kc, vc, None, slots, q_gain=gain, k_gain=gain)
            L.attention_causal(ctx, q_rot, kc.view(-1, hk, d)[:t], vc.view(-1, hk, d)[:t], o, cu, scale=d ** -0.5)
        L.attention_paged(ctx, q_rot, kc, vc, b, cu, lens, table, scale=d ** -0.5, max_q_len=t)
        ctx.sync()
        first = first or (a, b)
        assert torch.equal(a, first[0]) and torch.equal(c, first[0]) and torch.equal(b, first[1])
        # (half a step each of both kernels' numerators and outputs)
        assert (a.double() - b.double()).abs().max() <= 4 * R.half_step(BF16) * float(v.abs().max())


@pytest.mark.parametrize("q", [1, 90])
def test_paged_and_fused_calls_share_a_workspace(ctx, q):
    """The fused attention call stages its operands where the paged call keeps its parts."""
    from llmr_attn import configs as C
    from llmr_attn.runner import to_device
    dit = to_device(C.prepare(C.C3, L.rope_tables, seq_len=640, n_heads=2), out_dtype="f32")
    ctx.reserve(L.workspace_bytes(dit.desc()))
    p = Paged([q] * 3, [3000, 900, 20000], 8, 2, 128, 16, BF16, seed=q)
    want = p.check(ctx).clone()
    dit.run(ctx)
    ctx.sync()
    want_dit = dit.o.clone()
    for _ in range(15):
        p.o.fill_(7)
        dit.o.fill_(7)
        for _ in range(3):
            L.attention_paged(ctx, p.q, p.kc, p.vc, p.o, p.cu, p.kv, p.table, scale=p.d ** -0.5, max_q_len=q)
            dit.run(ctx)
        L.attention_paged(ctx, p.q, p.kc, p.vc, p.o, p.cu, p.kv, p.table, scale=p.d ** -0.5, max_q_len=q)
        ctx.sync()
        assert torch.equal(p.o, want) and torch.equal(dit.o, want_dit)
