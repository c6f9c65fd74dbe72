"""Workloads of the 4-bit KV cache and of the q/k-normed rotary append.

Three kinds of case, each one call as a serving program makes it:

  decode   one query row per sequence over a paged 4-bit cache (a generation step's attention)
  prefill  the newest n tokens of one sequence, causal, over a paged 4-bit cache (a prompt, a chunk of one, or
           the drafts of a speculative step)
  append   the projected q/k/v rows of new tokens: bias, RMS norm of every q and k head, rotary position and the
           write into the paged cache (f32, bf16 or 4-bit), then the rows read back as the values the cache holds

`run` computes them in plain torch where `own` is false and calls the package where it is true; `exact` gives the
values in 64 bits.

The 4-bit format: the 128 values of a (token, kv head) row in four groups of 32.  With x the group,
  scale = f16(bf16((max x - min x) / 15)),  offset = f16(min x + 8 scale),
  code = clamp(rint((x - offset) / scale) + 8, 0, 15)  (8 where scale = 0),
and the row stands for offset + (code - 8) * scale.
"""
import math
import random

import torch

own = False

D, PAGE = 128, 16
DEV = "cuda"
EPS = 1e-6


# ------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # a chat with one user: a 7B shape, 512 cached tokens and the new one; latency counts
        dict(name="decode one sequence", op="decode", heads=28, kv=4, batch=1, lo=513, hi=513),
        # a served batch of 64 requests of mixed age, shuffled pages
        dict(name="decode served batch", op="decode", heads=28, kv=4, batch=64, lo=1024, hi=8192),
        # long documents on an 8B shape
        dict(name="decode long context", op="decode", heads=32, kv=8, batch=8, lo=32768, hi=32768),
        # a 32B shape, odd batch, short and odd lengths, slots that hold nothing yet
        dict(name="decode short ragged", op="decode", heads=40, kv=8, batch=17, lo=0, hi=1999),
        # one rank of a tensor-parallel group (one kv head), one very long sequence
        dict(name="decode one kv head", op="decode", heads=8, kv=1, batch=1, lo=100003, hi=100003),
        # a whole prompt
        dict(name="prefill prompt", op="prefill", heads=28, kv=4, n=4096, prefix=0),
        # a chunk of a prompt behind a long prefix, odd sizes
        dict(name="prefill chunk", op="prefill", heads=32, kv=8, n=333, prefix=9001),
        # seven drafted tokens to verify
        dict(name="prefill drafts", op="prefill", heads=40, kv=8, n=7, prefix=2500),
        # one new token of one sequence, bf16 cache
        dict(name="append one token", op="append", heads=28, kv=4, seqs=1, n=1, start=512, cache="bf16", rows="f32",
             variant="interleaved", theta=1e6, bias=False),
        # the new tokens of a served batch into the 4-bit cache
        dict(name="append served batch", op="append", heads=32, kv=8, seqs=64, n=1, start=8191, cache="q4",
             rows="f32", variant="split_half", theta=5e5, bias=False),
        # a whole prompt into the 4-bit cache
        dict(name="append prompt", op="append", heads=28, kv=4, seqs=1, n=4096, start=0, cache="q4", rows="bf16",
             variant="interleaved", theta=1e6, bias=False),
        # drafted tokens of five requests, biased projections, f32 cache
        dict(name="append drafts", op="append", heads=40, kv=8, seqs=5, n=37, start=1001, cache="f32", rows="f32",
             variant="split_half", theta=1e6, bias=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(max(lo, 0.6)), math.log(hi)))))))


def draw(rng):
    heads, kv = rng.choice([(28, 4), (32, 8), (40, 8), (8, 1), (6, 3), (4, 4), (35, 7)])
    op = rng.choice(["decode", "prefill", "append"])
    if op == "decode":
        batch = _log(rng, 1, 64)
        hi = _log(rng, 1, min(131072, 8 * 32768 * 8 // (kv * batch)))
        return dict(op=op, heads=heads, kv=kv, batch=batch, lo=rng.randint(0, hi), hi=hi)
    if op == "prefill":
        n = _log(rng, 1, 4000)
        prefix = _log(rng, 0, 32000)
        most = 28 * 4096 * 4096 // (heads * n)  # the listed prompt's scores at most
        return dict(op=op, heads=heads, kv=kv, n=n, prefix=max(0, min(prefix, most - n)))
    seqs = _log(rng, 1, 64)
    n = _log(rng, 1, 4096 // seqs)
    return dict(op=op, heads=heads, kv=kv, seqs=seqs, n=n, start=_log(rng, 0, 16000),
                cache=rng.choice(["q4", "q4", "bf16", "f32"]), rows=rng.choice(["f32", "bf16"]),
                variant=rng.choice(["split_half", "interleaved"]), theta=rng.choice([1e6, 5e5]),
                bias=rng.random() < 0.5)


def _lens(case):
    """The cached lengths of a decode case's sequences: they belong to the case, so that its work is known."""
    r = random.Random("%(heads)d %(kv)d %(batch)d %(lo)d %(hi)d" % case)
    return [r.randint(case["lo"], case["hi"]) for _ in range(case["batch"])]


def _starts(case):
    """Where each sequence of an append case stands."""
    r = random.Random("%(seqs)d %(n)d %(start)d" % case)
    return [r.randint(case["start"] // 2, case["start"]) for _ in range(case["seqs"])]


def work(case):
    hq, hkv = case["heads"], case["kv"]
    row = {"q4": 80, "bf16": 256, "f32": 512}  # bytes of a cached K (or V) row of one kv head
    if case["op"] == "decode":
        tokens, rows = sum(_lens(case)), case["batch"]
        return {"bytes": tokens * hkv * 2 * row["q4"] + rows * hq * (2 * D + 1) * 4, "flops": 4 * tokens * hq * D}
    if case["op"] == "prefill":
        n, p = case["n"], case["prefix"]
        pairs = n * p + n * (n + 1) // 2
        return {"bytes": (p + n) * hkv * 2 * row["q4"] + n * hq * D * 4, "flops": 4 * pairs * hq * D}
    t = case["seqs"] * case["n"]
    es = 2 if case["rows"] == "bf16" else 4
    out = 4 if case["cache"] == "f32" else 2
    return {"bytes": t * D * (hq * 2 * es + 2 * hkv * (es + out)) + t * hkv * 2 * row[case["cache"]],
            "flops": t * (hq + hkv) * D * 10}


# ------------------------------------------------------------------------------------------------- inputs
def _quantize(x):
    """Codes [.., 128] (whole numbers 0..15) and f16 scale, offset [.., 4] of rows x [.., 128]."""
    g = x.float().unflatten(-1, (4, 32))
    lo, hi = g.amin(-1), g.amax(-1)
    scale = ((hi - lo) / 15).bfloat16().half()
    offset = (lo + 8 * scale.float()).half()
    s, o = scale.float().unsqueeze(-1), offset.float().unsqueeze(-1)
    c = torch.where(s > 0, ((g - o) / s).round() + 8, 8.0).clamp(0, 15)
    return c.flatten(-2).to(torch.uint8), scale, offset


def _cache(gen, lens, kv, keep_rows):
    """A paged 4-bit cache of `lens` tokens per sequence in shuffled pages.  Keys have channels of unlike size, as
    keys have; the slots behind a sequence's last token hold what an earlier owner of the page left there."""
    pages = [max(1, -(-n // PAGE)) for n in lens]
    most, total = max(pages), sum(pages)
    perm = torch.randperm(total, generator=gen, device=DEV)
    # the table, short rows filled with any page: the slots past a length are never looked at
    first = torch.tensor([0] + pages, device=DEV).cumsum(0)[:-1]
    at = first[:, None] + torch.arange(most, device=DEV)[None].clamp(max=total - 1)
    used = torch.arange(most, device=DEV)[None] < torch.tensor(pages, device=DEV)[:, None]
    table = torch.where(used, perm[at.clamp(max=total - 1)], perm[0])
    chan = torch.exp(0.5 * torch.randn(kv, 1, D, generator=gen, device=DEV))
    pool = {}
    for part in "kv":
        x = torch.randn(total, kv, PAGE, D, generator=gen, device=DEV)
        x = (x * chan if part == "k" else x).bfloat16()
        pool[part + "rows"] = x if keep_rows else None
        if not keep_rows:
            c, pool[part + "scale"], pool[part + "offset"] = _quantize(x)
            pool[part] = c[..., 0::2] | (c[..., 1::2] << 4)  # two codes to the byte, even channel low
        del x
    return table, pages, pool


def _engine(case, kv_dtype, pages, longest, variant="interleaved", theta=1e6):
    from oomllama_b200 import TurboConfig, TurboEngine

    cfg = TurboConfig(n_layers=1, hidden_size=case["heads"] * D, n_heads=case["heads"], n_kv_heads=case["kv"],
                      max_seq_len=longest, max_seqs=len(pages), n_pages=sum(pages), kv_dtype=kv_dtype,
                      rope_variant=variant, rope_theta=theta)
    return TurboEngine(cfg, device=torch.cuda.current_device(), assign_pages=False)


def _filled_engine(case, lens, table, pages, pool):
    """An engine whose cache was filled by the calls that a program makes."""
    e = _engine(case, "q4", pages, max(pages) * PAGE)
    for s, n in enumerate(lens):
        ids = table[s, :pages[s]]
        e.set_block_table(s, ids.tolist())
        if n:
            k, v = (pool[p][ids].transpose(1, 2).reshape(-1, case["kv"], D)[:n].contiguous() for p in ("krows", "vrows"))
            e.kv_write(0, s, k, v)
    return e


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    hq, hkv = case["heads"], case["kv"]
    st = {"case": case}
    if case["op"] in ("decode", "prefill"):
        lens = _lens(case) if case["op"] == "decode" else [case["prefix"] + case["n"]]
        table, pages, pool = _cache(gen, lens, hkv, own)
        if case["op"] == "decode":
            st["q"] = torch.randn(len(lens), hq, D, generator=gen, device=DEV)
        else:
            st["q"] = torch.randn(case["n"], hq, D, generator=gen, device=DEV).bfloat16()
        if own:
            st["engine"] = _filled_engine(case, lens, table, pages, pool)
            st["seqs"] = list(range(len(lens)))
        else:
            st.update(pool, table=table, lens=torch.tensor(lens, device=DEV))
        return st
    t, starts = case["seqs"] * case["n"], _starts(case)
    dt = torch.bfloat16 if case["rows"] == "bf16" else torch.float32
    rnd = lambda *shape, scale=1.0: scale * torch.randn(*shape, generator=gen, device=DEV)  # noqa: E731
    st["q"], st["k"], st["v"] = (rnd(t, h * D, scale=1.5).to(dt) for h in (hq, hkv, hkv))
    st["bias"] = [rnd(h * D, scale=0.3) if case["bias"] else None for h in (hq, hkv, hkv)]
    st["norm"] = [1 + rnd(D, scale=0.1) for _ in range(2)]
    if own:
        longest = -(-(max(starts) + case["n"]) // PAGE) * PAGE
        pages = [longest // PAGE] * case["seqs"]
        e = st["engine"] = _engine(case, case["cache"], pages, longest, case["variant"], case["theta"])
        perm = torch.randperm(sum(pages), generator=gen, device=DEV).tolist()
        for s in range(case["seqs"]):
            e.set_block_table(s, perm[s * pages[0]:(s + 1) * pages[0]])
            e.set_seq_len(0, s, starts[s])
        st["seqs"], st["starts"] = list(range(case["seqs"])), starts
    else:
        st["pos"] = (torch.tensor(starts, device=DEV)[:, None] + torch.arange(case["n"], device=DEV)).flatten()
        st["cos"], st["sin"] = _rope_rows(case["theta"], int(st["pos"].max()) + 1)
    return st


def _rope_rows(theta, n):
    """cos and sin [n, 64] as the cache's table has them: angle = f32(pos) * f32(1 / theta^(2i/128)), in f32."""
    e = 2 * torch.arange(D // 2, dtype=torch.float32) / D
    inv = 1.0 / (torch.tensor(theta, dtype=torch.float64) ** e.double()).float()
    a = torch.arange(n, dtype=torch.float32)[:, None] * inv
    return a.double().cos().float().to(DEV), a.double().sin().float().to(DEV)


# ------------------------------------------------------------------------------------------------- the passes
def run(st):
    op = st["case"]["op"]
    if own:
        return {"decode": _own_decode, "prefill": _own_prefill, "append": _own_append}[op](st)
    return {"decode": _plain_decode, "prefill": _plain_prefill, "append": _plain_append}[op](st)


def _own_decode(st):
    return st["engine"].decode(0, st["seqs"], st["q"], with_lse=True)


def _own_prefill(st):
    return st["engine"].prefill(0, 0, st["q"], out_dtype=torch.bfloat16)


def _own_append(st):
    e, c = st["engine"], st["case"]
    q = e.rope_append(0, st["seqs"], st["q"], st["k"], st["v"], *st["bias"], q_out_dtype=st["q"].dtype,
                      q_norm=st["norm"][0], k_norm=st["norm"][1], eps=EPS, starts=st["starts"])
    k, v = e.kv_gather(0, st["seqs"], st["starts"], c["n"],
                       out_dtype=torch.float32 if c["cache"] == "f32" else torch.bfloat16)
    return q, k, v


def _values(st, part):
    """The rows [sequences, kv heads, tokens, 128] that the cache's pages stand for."""
    at = st["table"]
    b = st[part][at]
    c = torch.stack((b & 15, b >> 4), -1).flatten(-2).float().unflatten(-1, (4, 32))
    x = (st[part + "offset"][at].float().unsqueeze(-1) + (c - 8) * st[part + "scale"][at].float().unsqueeze(-1)).flatten(-2)
    return x.transpose(1, 2).flatten(2, 3)


def _plain_attend(q, k, v, seen):
    """q [b, kv, rows, 128], k and v [b, kv, tokens, 128], seen [b, 1, rows, tokens] or broadcast."""
    s = (q @ k.transpose(-1, -2)) * (1 / math.sqrt(D))
    s = torch.where(seen, s, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    total = p.sum(-1, keepdim=True)
    out = torch.where(total > 0, (p @ v) / total, 0.0)
    return out, (m + torch.log(total)).squeeze(-1)


def _plain_decode(st):
    c = st["case"]
    k, v = _values(st, "k"), _values(st, "v")
    seen = torch.arange(k.shape[2], device=DEV) < st["lens"][:, None]
    q = st["q"].unflatten(1, (c["kv"], -1))
    out, lse = _plain_attend(q, k, v, seen[:, None, None])
    return out.flatten(1, 2), lse.flatten(1)


def _plain_prefill(st):
    c = st["case"]
    n, last = c["n"], c["prefix"] + c["n"]
    k, v = (_values(st, p)[:, :, :last] for p in "kv")
    q = st["q"].float().view(n, c["kv"], -1, D).permute(1, 2, 0, 3)
    seen = torch.arange(last, device=DEV) <= torch.arange(c["prefix"], last, device=DEV)[:, None]
    # one kv head's query heads side by side
    out, _ = _plain_attend(q, k[0].unsqueeze(1), v[0].unsqueeze(1), seen)
    return out.permute(2, 0, 1, 3).flatten(1, 2).bfloat16()


def _rotate(x, cos, sin, variant):
    """x [tokens, heads, 128], cos and sin [tokens, 64]."""
    cos, sin = cos.unsqueeze(1), sin.unsqueeze(1)
    if variant == "split_half":
        a, b = x[..., :D // 2], x[..., D // 2:]
        return torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)


def _normed(x, bias, weight, st, dt):
    x = x.to(dt).unflatten(-1, (-1, D))
    if bias is not None:
        x = x + bias.to(dt).view(1, -1, D)
    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.to(dt)
    return _rotate(x, st["cos"][st["pos"]].to(dt), st["sin"][st["pos"]].to(dt), st["case"]["variant"])


def _plain_append(st):
    c = st["case"]
    q = _normed(st["q"], st["bias"][0], st["norm"][0], st, torch.float32).to(st["q"].dtype)
    # keys in 64 bits: a code hangs on which side of a border a value lies
    k = _normed(st["k"], st["bias"][1], st["norm"][1], st, torch.float64).float()
    v = st["v"].float().unflatten(-1, (-1, D))
    if st["bias"][2] is not None:
        v = v + st["bias"][2].view(1, -1, D)
    if c["cache"] == "q4":
        k, v = _held(k), _held(v)
    out = torch.float32 if c["cache"] == "f32" else torch.bfloat16
    return q, k.to(out), v.to(out)


def _held(x):
    """The values that a 4-bit cache holds for rows x."""
    c, scale, offset = _quantize(x)
    g = c.float().unflatten(-1, (4, 32))
    return (offset.float().unsqueeze(-1) + (g - 8) * scale.float().unsqueeze(-1)).flatten(-2)


# ------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    hq, hkv = case["heads"], case["kv"]
    if case["op"] == "append":
        return _exact_append(case, st)
    lens = _lens(case) if case["op"] == "decode" else [case["prefix"] + case["n"]]
    outs, lses = [], []
    for s, n in enumerate(lens):
        if n == 0:
            outs.append(torch.zeros(1, hq, D, dtype=torch.float64, device=DEV))
            lses.append(torch.full((1, hq), -math.inf, dtype=torch.float64, device=DEV))
            continue
        ids = st["table"][s, :-(-n // PAGE)]
        k, v = _exact_rows(st, "k", ids)[:, :n], _exact_rows(st, "v", ids)[:, :n]
        q = (st["q"][s:s + 1] if case["op"] == "decode" else st["q"]).double()
        out, lse = torch.empty_like(q), torch.empty(q.shape[:2], dtype=torch.float64, device=DEV)
        ahead = None
        if case["op"] == "prefill":
            ahead = torch.ones(q.shape[0], n, dtype=torch.bool, device=DEV).triu(n - q.shape[0] + 1)
        for h in range(hq):
            z = torch.mv(k[h // (hq // hkv)], q[0, h])[None] if q.shape[0] == 1 else q[:, h] @ k[h // (hq // hkv)].T
            z = z / D ** 0.5
            if ahead is not None:
                z = z.masked_fill(ahead, -math.inf)
            lse[:, h] = torch.logsumexp(z, -1)
            out[:, h] = torch.softmax(z, -1) @ v[h // (hq // hkv)]
        outs.append(out)
        lses.append(lse)
    if case["op"] == "prefill":
        return outs[0]
    return torch.cat(outs), torch.cat(lses)


def _exact_rows(st, part, ids):
    """[kv heads, tokens, 128] of the pages `ids`, value by value from the format."""
    b = st[part][ids].permute(1, 0, 2, 3).flatten(1, 2).long()
    c = torch.empty(*b.shape[:2], D, dtype=torch.float64, device=DEV)
    c[..., 0::2], c[..., 1::2] = (b % 16).double(), (b // 16).double()
    s, o = (st[part + w][ids].permute(1, 0, 2, 3).flatten(1, 2).double().repeat_interleave(32, -1) for w in ("scale", "offset"))
    return o + s * (c - 8)


def _exact_append(case, st):
    """The rows with each pair turned as a complex number."""
    turn = torch.complex(st["cos"].double(), st["sin"].double())[st["pos"]][:, None]
    halves = case["variant"] == "split_half"
    rows = []
    for x, b, w in zip((st["q"], st["k"], st["v"]), st["bias"], (st["norm"][0], st["norm"][1], None)):
        x = x.double().view(x.shape[0], -1, D)
        if b is not None:
            x = x + b.double().view(-1, D)
        if w is not None:
            x = x * torch.rsqrt(x.pow(2).sum(-1, keepdim=True) / D + EPS) * w.double()
            pair = x.view(*x.shape[:2], 2, 64).transpose(-1, -2) if halves else x.view(*x.shape[:2], 64, 2)
            pair = torch.view_as_real(torch.complex(pair[..., 0], pair[..., 1]) * turn)
            x = (pair.transpose(-1, -2) if halves else pair).reshape(x.shape)
        rows.append(x)
    q, k, v = rows
    if case["cache"] == "q4":
        k, v = (_exact_held(x) for x in (k, v))
    return q, k, v


def _exact_held(x):
    g = x.view(*x.shape[:2], 4, 32)
    lo, hi = g.min(-1, keepdim=True).values, g.max(-1, keepdim=True).values
    scale = ((hi - lo) / 15).to(torch.bfloat16).to(torch.float16).double()
    offset = (lo + 8 * scale).to(torch.float16).double()
    c = torch.where(scale > 0, torch.round((g - offset) / scale), torch.zeros_like(g)).clamp(-8, 7)
    return (offset + c * scale).view(x.shape)
