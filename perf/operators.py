"""Measured cases of the paged-cache and sampling operators.

Three operators of a serving step: the append of new keys and values to a
paged cache (qk-norm and RoPE on the way), attention over that cache (decode
rows, speculative verify rows, prompt chunks; causal, or a sliding window with
a few first tokens that stay visible), and the verification of drafted tokens
against the target's probabilities from given random numbers.

``own`` selects the framework's kernels; otherwise ``run`` computes the same
with elementary torch operations.
"""
import math
import random

import torch

own = False

_DT = {"f16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------- cases


def listed():
    return [
        # a decode step's append: 8 sequences of the 8B shape, one row each
        dict(name="append_decode", op="append", batch=8, rows=1, ragged=False, ctx=640, H=32, Hkv=8, Dh=128, page=64,
             theta=5e5, norm=False, dtype="f16", shape=1),
        # the append of a batch of prompts of different lengths, hybrid model's heads with qk-norm
        dict(name="append_prompts", op="append", batch=16, rows=512, ragged=True, ctx=65536, H=24, Hkv=8, Dh=64,
             page=48, theta=1e6, norm=True, dtype="bf16", shape=2),
        # one user, early in a chat (the 1.1B shape): latency
        dict(name="decode_one", op="attention", batch=1, rows=1, ragged=False, ctx=257, spread=0, H=32, Hkv=4, Dh=64,
             page=16, window=0, sinks=0, dtype="f16", shape=3),
        # the verify rows of a speculative step with k = 4 (8B shape)
        dict(name="verify_rows", op="attention", batch=8, rows=5, ragged=False, ctx=4100, spread=1, H=32, Hkv=8,
             Dh=128, page=64, window=0, sinks=0, dtype="f16", shape=4),
        # continuous batching: 64 sequences of any length up to 16k
        dict(name="decode_ragged", op="attention", batch=64, rows=1, ragged=False, ctx=16384, spread=1, H=32, Hkv=8,
             Dh=128, page=64, window=0, sinks=0, dtype="f16", shape=5),
        # two users with very long contexts, small pages: split over the length
        dict(name="decode_long", op="attention", batch=2, rows=1, ragged=False, ctx=131071, spread=0, H=32, Hkv=8,
             Dh=128, page=16, window=0, sinks=0, dtype="bf16", shape=6),
        # streaming sessions: a window of 4096 and four sinks, the pages between freed
        dict(name="decode_window", op="attention", batch=32, rows=1, ragged=False, ctx=50000, spread=1, H=24, Hkv=8,
             Dh=64, page=32, window=4096, sinks=4, dtype="f16", shape=7),
        # a long prompt of the 8B shape: tensor bound
        dict(name="prompt_long", op="attention", batch=1, rows=8192, ragged=False, ctx=8192, spread=0, H=32, Hkv=8,
             Dh=128, page=64, window=0, sinks=0, dtype="f16", shape=8),
        # chunks of several prompts at once, windowed, next to earlier chunks
        dict(name="prompt_window", op="attention", batch=8, rows=777, ragged=True, ctx=3333, spread=1, H=24, Hkv=8,
             Dh=64, page=32, window=512, sinks=4, dtype="bf16", shape=9),
        # the draft's own sampled token (no drafts to verify), one small vocabulary
        dict(name="sample_draft", op="sample", batch=8, k=0, V=32000, temperature=0.8, noise=1.0, shape=10),
        # verification of four drafts for 8 sequences, the 8B shape's vocabulary
        dict(name="verify_drafts", op="sample", batch=8, k=4, V=128256, temperature=1.0, noise=0.5, shape=11),
        # the same for a large batch and an odd vocabulary shard
        dict(name="verify_many", op="sample", batch=61, k=5, V=65543, temperature=0.7, noise=0.25, shape=12),
    ]


def _logint(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "attention", "attention", "attention", "sample"])
    if op == "sample":
        k = rng.randint(0, 8)
        V = _logint(rng, 1000, 140000)
        batch = min(_logint(rng, 1, 96), max(1, 24_000_000 // ((2 * k + 1) * V)))
        return dict(op="sample", batch=batch, k=k, V=V, temperature=rng.choice([0.5, 0.7, 1.0, 1.3]),
                    noise=rng.choice([0.1, 0.5, 1.0]), shape=rng.randrange(1 << 30))
    Dh = rng.choice([64, 64, 128, 128, 256])
    Hkv = rng.choice([1, 2, 4, 8])
    H = Hkv * rng.choice([1, 2, 3, 4, 7, 8])
    page = rng.choice([16, 32, 48, 64, 128])
    dtype = rng.choice(["f16", "bf16"])
    shape = rng.randrange(1 << 30)
    if op == "append":
        batch = _logint(rng, 1, 64)
        rows = _logint(rng, 1, max(1, min(1000, 6000 // batch)))
        return dict(op="append", batch=batch, rows=rows, ragged=rng.random() < 0.5, ctx=rows + _logint(rng, 1, 60000),
                    H=H, Hkv=Hkv, Dh=Dh, page=page, theta=rng.choice([1e4, 5e5, 1e6]), norm=rng.random() < 0.5,
                    dtype=dtype, shape=shape)
    windowed = rng.random() < 0.4
    window = _logint(rng, 16, 5000) if windowed else 0
    sinks = rng.choice([0, 1, 4, 20]) if windowed else 0
    if rng.random() < 0.65:  # decode and verify rows
        batch = _logint(rng, 1, 128)
        rows = rng.choice([1, 1, 1, 2, 3, 5, 8])
        ctx = _logint(rng, 1, max(64, min(130000, 600_000_000 // (batch * Hkv * Dh * 4)))) + rows
    else:  # prompt chunks
        batch = rng.choice([1, 1, 2, 3, 5, 8])
        rows = _logint(rng, 17, max(32, 6000 // batch))
        ctx = rows + rng.choice([0, 0, _logint(rng, 1, 6000)])
    case = dict(op="attention", batch=batch, rows=rows, ragged=rng.random() < 0.5, ctx=ctx, spread=rng.choice([0, 1]),
                H=H, Hkv=Hkv, Dh=Dh, page=page, window=window, sinks=sinks, dtype=dtype, shape=shape)
    while work(case)["flops"] > 5e11:  # no larger than the listed prompt
        case["rows"] //= 2
        case["ctx"] //= 2
    return case


def _layout(case):
    """Row counts and first positions per sequence (from the case alone)."""
    rng = random.Random(case["shape"])
    B, rows, ctx = case["batch"], case["rows"], case["ctx"]
    counts, pos = [], []
    for b in range(B):
        n = rows
        if case["ragged"]:
            n = rows if b == 0 else rng.randint(0 if b % 5 == 4 else 1, rows)
        hi = ctx - n
        if case["op"] == "append":
            p = rng.randint(0, hi)
        elif case["spread"] and b:
            p = rng.randint(0, hi)
        else:
            p = hi
        counts.append(n)
        pos.append(p)
    return counts, pos


def _live(case, n, p):
    """The key ranges any of the rows p .. p + n - 1 sees: [(a, b), ...)."""
    end = p + n
    w = case.get("window", 0)
    if n == 0:
        return []
    if not w or p - w + 1 <= case["sinks"]:
        return [(0, end)]
    start = p - w + 1
    return ([(0, case["sinks"])] if case["sinks"] else []) + [(start, end)]


def work(case):
    """Bytes and flops of one pass: every input the rows need read once, the
    outputs written once."""
    if case["op"] == "sample":
        B, k, V = case["batch"], case["k"], case["V"]
        return {"bytes": (2 * k + 1) * B * V * 4 + B * k * 4 + 2 * B * (k + 1) * 4, "flops": (2 * k + 1) * B * V * 4}
    counts, pos = _layout(case)
    H, Hkv, Dh = case["H"], case["Hkv"], case["Dh"]
    rows = sum(counts)
    if case["op"] == "append":
        return {"bytes": rows * (H + 2 * Hkv) * Dh * 6, "flops": rows * (H + Hkv) * Dh * 4}
    keys = pairs = 0
    w, s = case["window"], case["sinks"]
    for n, p in zip(counts, pos):
        keys += sum(b - a for a, b in _live(case, n, p))
        for i in range(p, p + n):
            pairs += i + 1 if not w or i + 1 <= w else w + min(s, i + 1 - w)
    return {"bytes": keys * Hkv * Dh * 4 + rows * H * Dh * 4, "flops": 4 * pairs * H * Dh}


# ------------------------------------------------------------------ inputs


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1000003 + case["shape"] % 1000003)
    if case["op"] == "sample":
        return _prepare_sample(case, g)
    dt = _DT[case["dtype"]]
    counts, pos = _layout(case)
    B, H, Hkv, Dh, ps = case["batch"], case["H"], case["Hkv"], case["Dh"], case["page"]
    max_pages = (case["ctx"] + ps - 1) // ps
    # pages that hold a visible or newly written position, in shuffled order
    used = []
    for b, (n, p) in enumerate(zip(counts, pos)):
        live = [(p, p + n)] if case["op"] == "append" else _live(case, n, p)
        pages = sorted({i for a, e in live if e > a for i in range(a // ps, (e - 1) // ps + 1)})
        used += [(b, i) for i in pages]
    num_pages = len(used) + 3
    order = torch.randperm(num_pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((B, max_pages), -1, dtype=torch.int32, device="cuda")
    if used:
        ub = torch.tensor(used, device="cuda")
        table[ub[:, 0], ub[:, 1]] = order[:len(used)]
    k = torch.empty((num_pages, Hkv, ps, Dh), dtype=dt, device="cuda").normal_(generator=g)
    v = torch.empty_like(k).normal_(generator=g)
    rows = sum(counts)
    st = dict(case=case, counts=counts, first=pos, table=table, k=k, v=v,
              pos=torch.tensor(pos, dtype=torch.int32, device="cuda"))
    st["row_start"] = None
    if case["ragged"]:
        st["row_start"] = torch.tensor([0] + torch.tensor(counts).cumsum(0).tolist(), dtype=torch.int32, device="cuda")
    if case["op"] == "append":
        st["qkv"] = torch.randn((rows, (H + 2 * Hkv) * Dh), generator=g, device="cuda")
        st["q_norm"] = st["k_norm"] = None
        if case["norm"]:
            st["q_norm"] = torch.rand(Dh, generator=g, device="cuda") + 0.5
            st["k_norm"] = torch.rand(Dh, generator=g, device="cuda") + 0.5
    else:
        # queries as the append leaves them (scaled): scores of spread about 1.5
        st["q"] = (torch.randn((rows, H, Dh), generator=g, device="cuda") * (1.5 / math.sqrt(Dh))).to(dt)
    return st


def _prepare_sample(case, g):
    B, k, V = case["batch"], case["k"], case["V"]
    t = torch.randn((k + 1, B, V), generator=g, device="cuda") * 2.5
    st = dict(case=case, target=t, draft=None, drafts=None, u=torch.rand((B, k + 1), generator=g, device="cuda"))
    if k:
        d = t[:k] + case["noise"] * torch.randn((k, B, V), generator=g, device="cuda")
        # the draft sampled its tokens from its own probabilities
        c = torch.softmax(d.double() / case["temperature"], dim=2).cumsum(2)
        r = torch.rand((k, B, 1), generator=g, device="cuda").double() * c[..., -1:]
        st["drafts"] = (c <= r).sum(2).clamp_max(V - 1).to(torch.int32).t().contiguous()
        st["draft"] = d
    return st


# --------------------------------------------------------------------- run


def run(st):
    op = st["case"]["op"]
    if own:
        return _run_own(st, op)
    return {"append": _plain_append, "attention": _plain_attention, "sample": _plain_sample}[op](st)


def _run_own(st, op):
    from webgllm_b200 import paged, speculative

    c = st["case"]
    if op == "append":
        q = paged.rope_kv_paged(st["qkv"], st["pos"], st["k"], st["v"], st["table"], heads=c["H"], theta=c["theta"],
                                q_norm=st["q_norm"], k_norm=st["k_norm"], eps=1e-5, row_start=st["row_start"])
        return {"q": q, "k": st["k"], "v": st["v"]}
    if op == "attention":
        return {"out": paged.attention_paged(st["q"], st["pos"], st["k"], st["v"], st["table"], window=c["window"],
                                             sinks=c["sinks"], row_start=st["row_start"])}
    return {"picks": speculative.spec_sample(st["target"], st["draft"], st["drafts"], st["u"],
                                             temperature=c["temperature"])}


def _positions(st):
    """Sequence and position of every row."""
    n = torch.tensor(st["counts"], device="cuda")
    seq = torch.repeat_interleave(torch.arange(len(st["counts"]), device="cuda"), n)
    start = torch.cumsum(n, 0) - n
    return seq, st["pos"].long()[seq] + torch.arange(seq.numel(), device="cuda") - start[seq]


def _plain_append(st):
    c = st["case"]
    H, Hkv, Dh, ps = c["H"], c["Hkv"], c["Dh"], c["page"]
    seq, p = _positions(st)
    x = st["qkv"].view(-1, H + 2 * Hkv, Dh)
    q, k, v = x[:, :H], x[:, H:H + Hkv], x[:, H + Hkv:]
    if c["norm"]:
        q = q * torch.rsqrt((q * q).mean(2, keepdim=True) + 1e-5) * st["q_norm"]
        k = k * torch.rsqrt((k * k).mean(2, keepdim=True) + 1e-5) * st["k_norm"]
    # angles in 64 bits: positions reach far beyond what 32 bits resolve
    f = c["theta"] ** (-torch.arange(0, Dh, 2, device="cuda", dtype=torch.float64) / Dh)
    a = p.double()[:, None] * f
    cs, sn = torch.cos(a).float()[:, None], torch.sin(a).float()[:, None]

    def rot(t):
        lo, hi = t[..., :Dh // 2], t[..., Dh // 2:]
        return torch.cat([lo * cs - hi * sn, hi * cs + lo * sn], 2)

    dt = st["k"].dtype
    page = st["table"][seq, p // ps].long()
    st["k"][page, :, p % ps] = rot(k).to(dt)
    st["v"][page, :, p % ps] = v.to(dt)
    return {"q": (rot(q) / math.sqrt(Dh)).to(dt), "k": st["k"], "v": st["v"]}


def _plain_attention(st):
    c = st["case"]
    H, Hkv, Dh, ps, w, s = c["H"], c["Hkv"], c["Dh"], c["page"], c["window"], c["sinks"]
    out = torch.empty_like(st["q"])
    r = 0
    for b, (n, p) in enumerate(zip(st["counts"], st["first"])):
        if not n:
            continue
        j = torch.cat([torch.arange(a, e, device="cuda") for a, e in _live(c, n, p)])
        page = st["table"][b, j // ps].long()
        k = st["k"][page, :, j % ps].transpose(0, 1).float()  # [Hkv][keys][Dh]
        v = st["v"][page, :, j % ps].transpose(0, 1).float()
        i = torch.arange(p, p + n, device="cuda")[:, None]
        see = j <= i
        if w:
            see &= (j > i - w) | (j < s)
        q = st["q"][r:r + n].view(n, Hkv, H // Hkv, Dh).float()
        step = max(1, (1 << 29) // (H * j.numel()))
        for t in range(0, n, step):
            x = torch.einsum("nhgd,hkd->hgnk", q[t:t + step], k)
            x = x.masked_fill(~see[t:t + step], -math.inf)
            x = torch.exp(x - x.amax(3, keepdim=True))
            x = x / x.sum(3, keepdim=True)
            o = torch.einsum("hgnk,hkd->nhgd", x, v)
            out[r + t:r + t + o.shape[0]] = o.reshape(-1, H, Dh).to(out.dtype)
        r += n
    return {"out": out}


def _plain_sample(st):
    c = st["case"]
    B, k, V = c["batch"], c["k"], c["V"]
    # 64 bits throughout: the picks are decided by values next to a border
    p = torch.softmax(st["target"].double() / c["temperature"], 2)
    u = st["u"].double()
    n = torch.zeros(B, dtype=torch.long, device="cuda")
    bi = torch.arange(B, device="cuda")
    weight = p[k]
    if k:
        q = torch.softmax(st["draft"].double() / c["temperature"], 2)
        d = st["drafts"].long()
        pd = torch.gather(p[:k], 2, d.t()[:, :, None])[..., 0].t()
        qd = torch.gather(q, 2, d.t()[:, :, None])[..., 0].t()
        n = (u[:, :k] * qd < pd).long().cumprod(1).sum(1)
        q = torch.cat([q, torch.zeros_like(q[:1])])
        weight = (p[n, bi] - q[n, bi]).clamp_min(0)
    cum = weight.cumsum(1)
    tok = (cum <= u[:, k:k + 1] * cum[:, -1:]).sum(1).clamp_max(V - 1)
    picks = torch.full((k + 1, B), -1, dtype=torch.int32, device="cuda")
    for j in range(k):
        picks[j] = torch.where(j < n, st["drafts"][:, j], picks[j])
    picks[n, bi] = tok.to(torch.int32)
    return {"picks": picks}


# ------------------------------------------------------------------- exact


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(st, case)
    if case["op"] == "attention":
        return _exact_attention(st, case)
    return _exact_sample(st, case)


def _exact_append(st, case):
    H, Hkv, Dh, ps = case["H"], case["Hkv"], case["Dh"], case["page"]
    kp, vp = st["k"].double(), st["v"].double()
    x = st["qkv"].double().reshape(-1, H + 2 * Hkv, Dh)
    inv = torch.exp(torch.arange(Dh // 2, dtype=torch.float64, device="cuda") * (-2.0 * math.log(case["theta"]) / Dh))
    qs, r = [], 0
    for b, (n, p) in enumerate(zip(st["counts"], st["first"])):
        if not n:
            continue
        t = torch.arange(p, p + n, device="cuda")
        # a complex rotation of the pairs (j, j + Dh/2)
        z = torch.polar(torch.ones((n, 1, Dh // 2), dtype=torch.float64, device="cuda"), t[:, None, None] * inv)
        y = x[r:r + n]
        qk = y[:, :H + Hkv].clone()
        if case["norm"]:
            qk /= torch.sqrt(qk.square().mean(-1, keepdim=True) + 1e-5)
            qk[:, :H] *= st["q_norm"].double()
            qk[:, H:] *= st["k_norm"].double()
        zr = torch.complex(qk[..., :Dh // 2], qk[..., Dh // 2:]) * z
        qk = torch.cat([zr.real, zr.imag], -1)
        qs.append(qk[:, :H] * Dh ** -0.5)
        pages = st["table"][b].long()
        for i in range(p // ps, (p + n - 1) // ps + 1):
            lo, hi = max(p, i * ps), min(p + n, (i + 1) * ps)
            kp[pages[i], :, lo - i * ps:hi - i * ps] = qk[lo - p:hi - p, H:].transpose(0, 1)
            vp[pages[i], :, lo - i * ps:hi - i * ps] = y[lo - p:hi - p, H + Hkv:].transpose(0, 1)
        r += n
    return {"q": torch.cat(qs), "k": kp, "v": vp}


def _exact_attention(st, case):
    H, Hkv, Dh, ps = case["H"], case["Hkv"], case["Dh"], case["page"]
    w, s, G = case["window"], case["sinks"], case["H"] // case["Hkv"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    r = 0
    for b, (n, p) in enumerate(zip(st["counts"], st["first"])):
        if not n:
            continue
        nb = (p + n + ps - 1) // ps
        ids = st["table"][b, :nb].long()
        held = torch.nonzero(ids >= 0)[:, 0]
        at = (held[:, None] * ps + torch.arange(ps, device="cuda")).reshape(-1)  # positions of the held rows
        for h in range(Hkv):
            k = st["k"][ids[held], h].double().reshape(-1, Dh)
            v = st["v"][ids[held], h].double().reshape(-1, Dh)
            step = max(1, (1 << 27) // (G * at.numel()))
            for t in range(0, n, step):
                i = torch.arange(p + t, min(p + n, p + t + step), device="cuda")
                hide = at[None] > i[:, None]
                if w:
                    hide |= (at[None] <= i[:, None] - w) & (at[None] >= s)
                q = st["q"][r + t:r + t + i.numel(), h * G:(h + 1) * G].double()
                x = torch.softmax((q @ k.t()).masked_fill(hide[:, None], -math.inf), -1)
                out[r + t:r + t + i.numel(), h * G:(h + 1) * G] = x @ v
        r += n
    return {"out": out}


def _exact_sample(st, case):
    k, T = case["k"], case["temperature"]
    picks = torch.full((k + 1, case["batch"]), -1, dtype=torch.int32, device="cuda")

    def dist(row):
        x = row.double() / T
        e = torch.exp(x - x.max())
        return e / e.sum()

    for b in range(case["batch"]):
        n, left = 0, None
        u = [float(x) for x in st["u"][b].tolist()]
        while n < k:
            p, q, d = dist(st["target"][n, b]), dist(st["draft"][n, b]), int(st["drafts"][b, n])
            if not u[n] * float(q[d]) < float(p[d]):
                left = torch.clamp(p - q, min=0)
                break
            picks[n, b] = d
            n += 1
        if left is None:
            left = dist(st["target"][k, b])
        c = torch.cumsum(left, 0)
        i = int(torch.searchsorted(c, u[k] * c[-1], right=True))
        picks[n, b] = min(i, case["V"] - 1)
    return {"picks": picks}
